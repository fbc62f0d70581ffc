// Between h's gradient and x's in the gated feed-forward block: from d = dL/dh and
// the forward's float sums g and u, dL/dg = d u act'(g) and dL/du = d act(g), as operands of
// the products past the weights.  One T number for each would add its rounding to x's
// gradient, as large as that one's own (with both, 1.41 times the error of a float32 form), so
// each is two: the value rounded to T, and the rest rounded to T, together within 2^-16 of
// the value in bfloat16 and 2^-22 in float16.  The products then take twice the MFMAs.
//
// HBM-bound: 10 bytes read and 8 written per element.  Eight columns per thread.  dg and du
// lie side by side in a row, each padded with zeros to whole steps of 64 columns, then
// their rests.
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

// v rounded to T, and the rest; a value past T's range has no rest (inf - inf).
template <int DT>
struct Pair {
  float hi, lo;
  __device__ __forceinline__ explicit Pair(float v) {
    // the rounding may pass T's largest number, of which the rest is then taken
    hi = T16<DT>::to_f32(T16<DT>::round1(v));
    if (__builtin_isinf(hi) && !__builtin_isinf(v)) hi = __builtin_copysignf(kMost, v);
    lo = __builtin_isinf(hi) ? 0.f : v - hi;
  }
  static constexpr float kMost = DT == kBF16 ? 0x1.fep127f : 65504.f;
};

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
    u32x4 out[4];                               // dg, du, and their rests
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[4][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float a, da;
        act_grad(g[2 * q + e], act, a, da);
        const Pair<DT> x(dv[2 * q + e] * u[2 * q + e] * da), y(dv[2 * q + e] * a);
        v[0][e] = x.hi;
        v[1][e] = y.hi;
        v[2][e] = x.lo;
        v[3][e] = y.lo;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i][q] = T::pack2(v[i][0], v[i][1]);
    }
    uint16_t* row = dgu + m * 4 * P + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(row + i * P) = out[i];
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
