// Instantiations of the dense gated feed-forward block's kernels for one (dtype,
// bits, group size) triple, compiled once per triple; -fno-slp-vectorize as
// dense.hip has it.
#include "glu_wide.cuh"

#if !defined(MQ_INST_DT) || !defined(MQ_INST_BITS) || !defined(MQ_INST_GS)
#error "compile with -DMQ_INST_DT=<0|1> -DMQ_INST_BITS=<4|8> -DMQ_INST_GS=<32|64|128>"
#endif

namespace mq {
template struct GluSkinnyLaunch<MQ_INST_DT, MQ_INST_BITS, MQ_INST_GS>;
template struct GluWideLaunch<MQ_INST_DT, MQ_INST_BITS, MQ_INST_GS>;
}  // namespace mq
