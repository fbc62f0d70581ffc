// Instantiations of the products past quantized weights (qmm_grad.cuh) for one
// (dtype, bits, group size) triple, compiled once per triple;
// -fno-slp-vectorize as dense.hip has it.
#include "qmm_grad.cuh"

#if !defined(MQ_INST_DT) || !defined(MQ_INST_BITS) || !defined(MQ_INST_GS)
#error "compile with -DMQ_INST_DT=<0|1> -DMQ_INST_BITS=<4|8> -DMQ_INST_GS=<32|64|128>"
#endif

namespace mq {
template struct GradLaunch<MQ_INST_DT, MQ_INST_BITS, MQ_INST_GS>;
}  // namespace mq
