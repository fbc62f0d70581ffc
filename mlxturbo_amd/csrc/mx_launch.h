// Launchers of the MXFP4 kernels, called by the C ABI (abi.hip); each enqueues
// on the given stream and returns 0, a HIP error or kStatusUnsupported.
#pragma once
#include "launch.h"

namespace mq {

constexpr int kMxGroup = 32;                    // codes per scale

// (wq, scales) = the MXFP4 codes of w [N, K] (any of the three dtypes), and
// back (mx_formats.hip).
int launch_mx_quantize(const void* w, uint32_t* wq, uint8_t* scales, int64_t N, int64_t K,
                       int dtype, hipStream_t st);
int launch_mx_dequantize(const uint32_t* wq, const uint8_t* scales, void* out, int64_t N,
                         int64_t K, int dtype, hipStream_t st);

// out [M, N] = x [M, K] . deq(w)^T on the skinny kernel (mx_skinny.cuh); QQ: x
// brought into MXFP4 first.  Any M; *nlaunch counts the kernels enqueued.
template <int DT, bool QQ>
struct MxSkinnyLaunch {
  static int run(const void* x, const uint32_t* w, const uint8_t* s, void* out, int64_t M,
                 int64_t N, int64_t K, hipStream_t st, int* nlaunch);
};

// gather_qmm over P (x batch, expert) pairs on the skinny kernel; ws as
// gather_workspace_bytes(P, M) says.
template <int DT>
struct MxGatherLaunch {
  static int run(const void* x, const uint32_t* w, const uint8_t* s, const int32_t* lhs,
                 const int32_t* rhs, void* out, int64_t P, int64_t B, int64_t M, int64_t N,
                 int64_t K, int64_t E, void* ws, hipStream_t st, int* nlaunch);
};

}  // namespace mq
