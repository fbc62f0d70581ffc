// The skinny MXFP4 products of one dtype (MQ_INST_DT).
#include "mx_skinny.cuh"

namespace mq {
template struct MxSkinnyLaunch<MQ_INST_DT, false>;
template struct MxSkinnyLaunch<MQ_INST_DT, true>;
template struct MxGatherLaunch<MQ_INST_DT>;
}  // namespace mq
