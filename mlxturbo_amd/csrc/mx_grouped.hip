// gather_qmm of many pairs over MXFP4 banks, of one dtype (MQ_INST_DT).
#include "mx_grouped.cuh"

namespace mq {
template struct MxGroupedLaunch<MQ_INST_DT>;
}  // namespace mq
