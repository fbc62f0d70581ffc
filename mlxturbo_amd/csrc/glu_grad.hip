// Between h's gradient and x's in the gated feed-forward block: from d = dL/dh and
// the forward's float sums g and u, dL/dg = d u act'(g) and dL/du = d act(g), rounded
// to T for the products past the weights (their one rounding: g and u are float).
//
// HBM-bound: 10 bytes read and 4 written per element, 2048 x 17408 in 103 us, 4.8 TB/s.  Eight columns per thread.  The two
// halves lie side by side in a row, each padded with zeros to whole steps of 64
// columns.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "glu_launch.h"

namespace mq {

namespace {

// act(g) and its derivative.
__device__ __forceinline__ void act_grad(float g, int act, float& a, float& da) {
  const float gg = kGeluCubic * g * g;
  const float z = act == kActSilu ? g : kGeluZ * g * (1.0f + gg);
  const float s = 1.0f / (1.0f + expf(-z));
  a = g * s;
  // g s (1 - s) z' vanishes at both ends, where z' may be infinite
  const float dz = act == kActSilu ? 1.0f : fminf(kGeluZ * (1.0f + 3.0f * gg), 0x1p60f);
  da = s + a * (1.0f - s) * dz;
}

// Grid (ceil(P / 2048), min(M, 65535)), 256 threads; P = 64 ceil(N / 64).  VEC: N in
// whole eights, all arrays 16-byte aligned.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void glu_grad_kernel(const uint16_t* __restrict__ d,
                                                       const float* __restrict__ gf,
                                                       const float* __restrict__ uf,
                                                       uint16_t* __restrict__ dgu, int64_t M,
                                                       int64_t N, int64_t P, int act) {
  using T = T16<DT>;
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= P) return;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
    const int64_t o = m * N + c;
    float dv[8], g[8], u[8];
    if (VEC && c < N) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(d + o);
#pragma unroll
      for (int e = 0; e < 8; ++e) dv[e] = T::to_f32((uint16_t)(v[e / 2] >> (16 * (e & 1))));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(gf + o + 4 * q);
        const f32x4 b = *reinterpret_cast<const f32x4*>(uf + o + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[4 * q + e] = a[e];
          u[4 * q + e] = b[e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = c + e < N;
        dv[e] = in ? T::to_f32(d[o + e]) : 0.f;
        g[e] = in ? gf[o + e] : 0.f;
        u[e] = in ? uf[o + e] : 0.f;
      }
    }
    u32x4 og, ou;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float x[2], y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float a, da;
        act_grad(g[2 * q + e], act, a, da);
        x[e] = dv[2 * q + e] * u[2 * q + e] * da;
        y[e] = dv[2 * q + e] * a;
      }
      og[q] = T::pack2(x[0], x[1]);
      ou[q] = T::pack2(y[0], y[1]);
    }
    uint16_t* row = dgu + m * 2 * P + c;
    *reinterpret_cast<u32x4*>(row) = og;
    *reinterpret_cast<u32x4*>(row + P) = ou;
  }
}

// Rows of N elements to rows of P, zeros past N.
__global__ __launch_bounds__(256) void pad_rows_kernel(const uint16_t* __restrict__ d,
                                                       uint16_t* __restrict__ out, int64_t M,
                                                       int64_t N, int64_t P) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= P) return;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y)
    out[m * P + c] = c < N ? d[m * N + c] : (uint16_t)0;
}

inline unsigned grid_rows(int64_t M) { return (unsigned)(M < 65535 ? M : 65535); }

}  // namespace

int launch_glu_grad(const void* d, const float* gf, const float* uf, void* dgu, int64_t M,
                    int64_t N, int act, int dtype, hipStream_t st) {
  const int64_t P = 64 * grad_steps(N);
  const dim3 grid((unsigned)((P + 2047) / 2048), grid_rows(M));
  const bool vec = N % 8 == 0 && (((uintptr_t)d | (uintptr_t)gf | (uintptr_t)uf) & 15u) == 0;
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, (const uint16_t*)d, gf, uf, (uint16_t*)dgu, M,
                       N, P, act);
    return 0;
  };
  if (dtype == kBF16) return vec ? go(glu_grad_kernel<kBF16, true>) : go(glu_grad_kernel<kBF16, false>);
  return vec ? go(glu_grad_kernel<kF16, true>) : go(glu_grad_kernel<kF16, false>);
}

int launch_pad_rows(const void* d, void* out, int64_t M, int64_t N, hipStream_t st) {
  const int64_t P = 64 * grad_steps(N);
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)((P + 255) / 256), grid_rows(M)), dim3(256),
                     0, st, (const uint16_t*)d, (uint16_t*)out, M, N, P);
  return 0;
}

}  // namespace mq
