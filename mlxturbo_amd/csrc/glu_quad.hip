// The gated feed-forward block of one row: instantiations of the quad kernel's gated form
// (qmv_quad.cuh) for one (dtype, bits) pair and every group size, compiled as quad.hip is.
#include "qmv_quad.cuh"

#if !defined(MQ_INST_DT) || !defined(MQ_INST_BITS)
#error "compile with -DMQ_INST_DT=<0|1> -DMQ_INST_BITS=<4|8>"
#endif

namespace mq {

template struct GluQuadLaunch<MQ_INST_DT, MQ_INST_BITS, 32>;
template struct GluQuadLaunch<MQ_INST_DT, MQ_INST_BITS, 64>;
template struct GluQuadLaunch<MQ_INST_DT, MQ_INST_BITS, 128>;

}  // namespace mq
