// Between h's gradient and x's in the gated feed-forward block: from d = dL/dh and
// the forward's float sums g and u, dL/dg = d u act'(g) and dL/du = d act(g), as operands of
// the products past the weights.  One T number for each would add its rounding to x's
// gradient, as large as that one's own (with both, 1.41 times the error of a float32 form), so
// each is two: the value rounded to T, and the rest rounded to T, together within 2^-16 of
// the value in bfloat16 and 2^-22 in float16.  The products then take twice the MFMAs.
//
// float16 holds no more than 65504, and d u act'(g) of a scaled loss may pass it where x's
// gradient does not.  Its rows are multiplied by a power of two that brings their largest
// value to 2^14 .. 2^15, which the product's sums are divided by: exact, and what falls below
// float16's smallest number is then below 2^-39 of the row's largest.
//
// HBM-bound: 10 bytes read and 8 written per element, 2048 x 17408 in 119 us, 5.4 TB/s; float16,
// 301 x 8192, 20 us, of which the second computation and the wait between are half (9.3
// unscaled).  Eight columns per thread.  dg and du
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

// dg and du of columns c .. c + 7 of row m, zeros past N.  VEC: N in whole eights, all
// arrays 16-byte aligned.
template <int DT, bool VEC>
__device__ __forceinline__ void row_values(const uint16_t* __restrict__ d,
                                           const float* __restrict__ gf,
                                           const float* __restrict__ uf, int64_t m, int64_t c,
                                           int64_t N, int act, float (&x)[8], float (&y)[8]) {
  using T = T16<DT>;
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
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float a, da;
    act_grad(g[e], act, a, da);
    x[e] = dv[e] * u[e] * da;
    y[e] = dv[e] * a;
  }
}

// Their pairs to a row of dgu, from its column c on.
template <int DT>
__device__ __forceinline__ void put_pairs(uint16_t* row, int64_t P, const float (&x)[8],
                                          const float (&y)[8]) {
  u32x4 out[4];                                 // dg, du, and their rests
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const Pair<DT> x0(x[2 * q]), x1(x[2 * q + 1]), y0(y[2 * q]), y1(y[2 * q + 1]);
    out[0][q] = T16<DT>::pack2(x0.hi, x1.hi);
    out[1][q] = T16<DT>::pack2(y0.hi, y1.hi);
    out[2][q] = T16<DT>::pack2(x0.lo, x1.lo);
    out[3][q] = T16<DT>::pack2(y0.lo, y1.lo);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(row + i * P) = out[i];
}

// bfloat16.  Grid (ceil(P / 2048), min(M, 65535)), 256 threads; P = 64 ceil(N / 64).
template <bool VEC>
__global__ __launch_bounds__(256) void glu_grad_kernel(const uint16_t* __restrict__ d,
                                                       const float* __restrict__ gf,
                                                       const float* __restrict__ uf,
                                                       uint16_t* __restrict__ dgu, int64_t M,
                                                       int64_t N, int64_t P, int act) {
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= P) return;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
    float x[8], y[8];
    row_values<kBF16, VEC>(d, gf, uf, m, c, N, act, x, y);
    put_pairs<kBF16>(dgu + m * 4 * P + c, P, x, y);
  }
}

constexpr int kRowThreads = 512;

// float16: a row per workgroup, computed twice, for its largest value and for its pairs (the
// second time from the L2 or the cache behind it).  undo[m]: the power of two that the sums
// of row m are multiplied by.  Infinities and NaN stay, and the finite values set the factor.
template <bool VEC>
__global__ __launch_bounds__(kRowThreads) void glu_grad_scaled_kernel(
    const uint16_t* __restrict__ d, const float* __restrict__ gf, const float* __restrict__ uf,
    uint16_t* __restrict__ dgu, float* __restrict__ undo, int64_t M, int64_t N, int64_t P,
    int act) {
  __shared__ uint32_t tops[kRowThreads / 64];
  const int t = threadIdx.x;
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
    float x[8], y[8];
    uint32_t top = 0;                           // bits of the largest magnitude
    for (int64_t c = 8 * t; c < N; c += 8 * kRowThreads) {
      row_values<kF16, VEC>(d, gf, uf, m, c, N, act, x, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t a = __float_as_uint(x[e]) & 0x7fffffffu;
        const uint32_t b = __float_as_uint(y[e]) & 0x7fffffffu;
        if (a < 0x7f800000u) top = max(top, a);
        if (b < 0x7f800000u) top = max(top, b);
      }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if ((t & 63) == 0) tops[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowThreads / 64; ++w) top = max(top, tops[w]);
    __syncthreads();
    // largest in [2^e, 2^(e + 1)): times 2^(14 - e); both factors stay normal numbers
    const int e = (int)(top >> 23) - 127, k = top ? min(14 - e, 126) : 0;
    const float factor = __uint_as_float((uint32_t)(127 + k) << 23);
    if (t == 0) undo[m] = __uint_as_float((uint32_t)(127 - k) << 23);
    for (int64_t c = 8 * t; c < P; c += 8 * kRowThreads) {
      row_values<kF16, VEC>(d, gf, uf, m, c, N, act, x, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= factor;
        y[i] *= factor;
      }
      put_pairs<kF16>(dgu + m * 4 * P + c, P, x, y);
    }
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

int launch_glu_grad(const void* d, const float* gf, const float* uf, void* dgu, float* undo,
                    int64_t M, int64_t N, int act, int dtype, hipStream_t st) {
  const int64_t P = 64 * grad_steps(N);
  const bool vec = N % 8 == 0 && (((uintptr_t)d | (uintptr_t)gf | (uintptr_t)uf) & 15u) == 0;
  if (dtype == kBF16) {
    const dim3 grid((unsigned)((P + 2047) / 2048), grid_rows(M));
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, (const uint16_t*)d, gf, uf, (uint16_t*)dgu,
                         M, N, P, act);
    };
    if (vec) go(glu_grad_kernel<true>);
    else go(glu_grad_kernel<false>);
  } else {
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3(grid_rows(M)), dim3(kRowThreads), 0, st, (const uint16_t*)d, gf,
                         uf, (uint16_t*)dgu, undo, M, N, P, act);
    };
    if (vec) go(glu_grad_scaled_kernel<true>);
    else go(glu_grad_scaled_kernel<false>);
  }
  return 0;
}

int launch_pad_rows(const void* d, void* out, int64_t M, int64_t N, hipStream_t st) {
  const int64_t P = 64 * grad_steps(N);
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)((P + 255) / 256), grid_rows(M)), dim3(256),
                     0, st, (const uint16_t*)d, (uint16_t*)out, M, N, P);
  return 0;
}

}  // namespace mq
