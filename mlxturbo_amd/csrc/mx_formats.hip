// MXFP4 quantize and dequantize (format and conversions: mx_common.cuh).
//
// Bound by memory: 2 or 4 bytes per value on one side and 0.53 on the other.
// A thread takes 8 values of a group, so a 16-bit type moves 16 bytes per load
// and a wave whole kilobytes; the four threads of a group agree on its scale
// over two DPP exchanges.  kMxUnits units of 8 values per thread, a
// workgroup's units contiguous, all loads issued before the first use.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx_common.cuh"
#include "mx_launch.h"

namespace mq {

namespace {

constexpr int kMxThreads = 256;
constexpr int kMxUnits = 4;

// units: N * K / 8, a multiple of 4, so a group's four threads are all there
// or none is.
template <int DT>
__global__ __launch_bounds__(kMxThreads) void mx_quantize_kernel(const void* __restrict__ w,
                                                                 uint32_t* __restrict__ wq,
                                                                 uint8_t* __restrict__ scales,
                                                                 int64_t units) {
  constexpr int R = DT == kF32 ? 2 : 1;         // 16-byte loads per unit
  const int64_t u0 = (int64_t)blockIdx.x * (kMxThreads * kMxUnits) + threadIdx.x;
  u32x4 v[kMxUnits][R];
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    const int64_t u = u0 + i * kMxThreads;
    if (u >= units) continue;
#pragma unroll
    for (int r = 0; r < R; ++r) v[i][r] = reinterpret_cast<const u32x4*>(w)[u * R + r];
  }
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    const int64_t u = u0 + i * kMxThreads;
    if (u >= units) continue;
    uint32_t top = 0;
    if constexpr (DT == kF32) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, v[i][r][j] & 0x7fffffffu);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) top = mx_max2(top, v[i][0][j] & 0x7fff7fffu);
      top = max(top & 0xffffu, top >> 16);
    }
    const uint32_t e = mx_scale_byte<DT>(mx_quad_max(top));
    const float s = mx_scale(e);
    uint32_t c;
    if constexpr (DT == kF32) {
      auto f = [&](int j) { return __uint_as_float(v[i][j >> 2][j & 3]); };
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f(0), f(1), s, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(2), f(3), s, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(4), f(5), s, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(6), f(7), s, 3);
    } else {
      c = mx_code_word<DT>(v[i][0], s);
    }
    wq[u] = e == 255 ? 0u : c;
    if ((u & 3) == 0) scales[u >> 2] = (uint8_t)e;
  }
}

template <int DT>
__global__ __launch_bounds__(kMxThreads) void mx_dequantize_kernel(
    const uint32_t* __restrict__ wq, const uint8_t* __restrict__ scales, void* __restrict__ out,
    int64_t units) {
  const int64_t u0 = (int64_t)blockIdx.x * (kMxThreads * kMxUnits) + threadIdx.x;
  uint32_t c[kMxUnits], e[kMxUnits];
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    const int64_t u = u0 + i * kMxThreads;
    if (u >= units) continue;
    c[i] = wq[u];
    e[i] = scales[u >> 2];
  }
#pragma unroll
  for (int i = 0; i < kMxUnits; ++i) {
    const int64_t u = u0 + i * kMxThreads;
    if (u >= units) continue;
    const float s = mx_scale(e[i]);
    if constexpr (DT == kF32) {
      const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 0);
      const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 1);
      const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 2);
      const f32x2 f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], s, 3);
      f32x4* o = reinterpret_cast<f32x4*>(out) + u * 2;
      o[0] = (f32x4){a.x, a.y, b.x, b.y};
      o[1] = (f32x4){d.x, d.y, f.x, f.y};
    } else {
      reinterpret_cast<u32x4*>(out)[u] = mx_word<DT>(c[i], s);
    }
  }
}

inline int64_t mx_blocks(int64_t units) {
  return (units + kMxThreads * kMxUnits - 1) / (kMxThreads * kMxUnits);
}

}  // namespace

int launch_mx_quantize(const void* w, uint32_t* wq, uint8_t* scales, int64_t N, int64_t K,
                       int dtype, hipStream_t st) {
  const int64_t units = N * (K / 8), nb = mx_blocks(units);
  if (!mx_grid_ok(nb, kMxThreads)) return kStatusUnsupported;
#define MQ_MXQ(DT)                                                                            \
  hipLaunchKernelGGL(mx_quantize_kernel<DT>, dim3((unsigned)nb), dim3(kMxThreads), 0, st, w, wq, \
                     scales, units)
  if (dtype == kBF16) MQ_MXQ(kBF16);
  else if (dtype == kF16) MQ_MXQ(kF16);
  else MQ_MXQ(kF32);
#undef MQ_MXQ
  return 0;
}

int launch_mx_dequantize(const uint32_t* wq, const uint8_t* scales, void* out, int64_t N,
                         int64_t K, int dtype, hipStream_t st) {
  const int64_t units = N * (K / 8), nb = mx_blocks(units);
  if (!mx_grid_ok(nb, kMxThreads)) return kStatusUnsupported;
#define MQ_MXD(DT)                                                                              \
  hipLaunchKernelGGL(mx_dequantize_kernel<DT>, dim3((unsigned)nb), dim3(kMxThreads), 0, st, wq, \
                     scales, out, units)
  if (dtype == kBF16) MQ_MXD(kBF16);
  else if (dtype == kF16) MQ_MXD(kF16);
  else MQ_MXD(kF32);
#undef MQ_MXD
  return 0;
}

}  // namespace mq
