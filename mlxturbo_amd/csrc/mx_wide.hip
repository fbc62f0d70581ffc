// The wide MXFP4 products of one dtype (MQ_INST_DT), T or 4-bit x (MQ_INST_QQ).
#include "mx_wide.cuh"

namespace mq {
template struct MxWideLaunch<MQ_INST_DT, MQ_INST_QQ>;
}  // namespace mq
