// Products of few x rows with MXFP4 weights: the weight stream bounds them.
//
// out[m, n] = sum over groups g of 32 codes of 2^(e[n, g] - 127) *
// (x[m, g] . code[n, g]), summed in float by MFMAs of 16x16x32 over the
// weights' T values (T(code * 2^(e - 127))), or, QQ, of 16x16x128 over the
// codes of both operands with their scale bytes.
//
// A wave owns 16 NT weight rows and a slice of K; the KW waves of a workgroup
// split K and add their sums through LDS in wave order, so a row's result
// depends on N and K alone, not on how many rows the call has.  Per step of
// 128 codes lane (r = lane & 15, c = lane >> 4) takes the 16 bytes of row r
// that hold the step's group c, all of one scale, and the matching 64 bytes of
// x row r; MFMA j multiplies codes 8 j .. 8 j + 7 of every lane's group (the
// order of k within a step is the same on both sides, so it does not matter).
// Weights and x go straight to registers, D steps ahead; the tile's scale
// bytes are one contiguous block, copied to LDS first.
//
// Groups past K: zero codes (outside the buffer range), scale byte 0 and x from
// a block of zeros, so no 0 * inf arises.  Rows of x past M read row 0 of the
// tile; their columns are not stored.
#pragma once
#include "mx_common.cuh"
#include "mx_launch.h"

namespace mq {

__device__ __align__(64) static const unsigned char mx_zeros[64] = {};

// Dynamic LDS: scales of 16 NT rows, later the waves' sums.
template <int MT, int NT, int KW>
__host__ __device__ inline size_t mx_skinny_lds(int64_t G) {
  const size_t sc = ((size_t)(16 * NT) * (size_t)G + 16 + 15) & ~(size_t)15;
  const size_t red = (size_t)KW * NT * MT * 1024;
  return sc > red ? sc : red;
}

// xp[i]: x row of tile row 16 i + r, at the lane's 64 bytes of step 0 (+ 32 c
// values).  w, scales: the tile's first row; nrows <= 16 NT of them exist.
// put(t, i, l, v): v[q] = the sum of weight row 16 t + 4 (l >> 4) + q and x
// row 16 i + (l & 15).
template <int DT, bool QQ, int MT, int NT, int KW, class Put>
__device__ __forceinline__ void mx_skinny_tile(const unsigned char* const (&xp)[MT],
                                               const uint32_t* __restrict__ w,
                                               const uint8_t* __restrict__ scales, int nrows,
                                               int G, unsigned char* __restrict__ lds, Put put) {
  constexpr int D = MT == 1 ? 4 : 2;            // steps in flight
  constexpr int NTHR = 64 * KW;
  using T = T16<DT>;
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int S = (G + 3) >> 2, per = (S + KW - 1) / KW;
  const int s0 = min(S, wave * per), s1 = min(S, s0 + per);
  const auto rw = wide_rsrc(w, (int64_t)nrows * G * 16);
  uint32_t skew;
  const auto rs = mx_scale_rsrc(scales, (int64_t)nrows * G, skew);
  const uint32_t sbytes = (uint32_t)(nrows * G) + skew;

  uint32_t wo[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) wo[j] = (uint32_t)((16 * j + r) * G + c) * 16u;
  u32x4 W[D][NT], X[D][MT][4];
  auto ok = [&](int s) { return s < s1 && 4 * s + c < G; };
  auto load = [&](int d, int s) {
    const bool v = ok(s);
#pragma unroll
    for (int j = 0; j < NT; ++j)
      W[d][j] = __builtin_amdgcn_raw_buffer_load_b128(rw, v ? wo[j] + 64u * (uint32_t)s : 0x80000000u,
                                                      0, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const u32x4* a = reinterpret_cast<const u32x4*>(v ? xp[i] + 256 * (int64_t)s : mx_zeros);
#pragma unroll
      for (int j = 0; j < 4; ++j) X[d][i][j] = a[j];
    }
  };
  // the first scale pieces go out before the weights
  u32x4 sv[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    sv[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (uint32_t)(i * NTHR + t) * 16u, 0, 0);
#pragma unroll
  for (int d = 0; d < D; ++d) load(d, s0 + d);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t o = (uint32_t)(i * NTHR + t) * 16u;
    if (o < sbytes) *reinterpret_cast<u32x4*>(lds + o) = sv[i];
  }
  for (uint32_t o = (uint32_t)(2 * NTHR + t) * 16u; o < sbytes; o += NTHR * 16u)
    *reinterpret_cast<u32x4*>(lds + o) = __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0);
  __syncthreads();

  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // rows past the tile's last read its scales
  uint32_t so[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) so[j] = skew + (uint32_t)(min(16 * j + r, nrows - 1) * G + c);

  for (int s = s0; s < s1; s += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const bool v = ok(s + d);
      uint32_t e[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint32_t b = lds[v ? so[j] + 4u * (uint32_t)(s + d) : skew];
        e[j] = v ? b : 0u;
      }
      if constexpr (QQ) {
        i32x8 xq[MT];
        uint32_t xe[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t top = 0;
#pragma unroll
          for (int q = 0; q < 16; ++q) top = mx_max2(top, X[d][i][q >> 2][q & 3] & 0x7fff7fffu);
          xe[i] = mx_scale_byte<DT>(max(top & 0xffffu, top >> 16));
          const float xs = mx_scale(xe[i]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t cw = mx_code_word<DT>(X[d][i][q], xs);
            xq[i][q] = (int)(xe[i] == 255 ? 0u : cw);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const i32x8 a = __builtin_shufflevector(bitcast<i32x4>(W[d][j]), bitcast<i32x4>(W[d][j]),
                                                  0, 1, 2, 3, -1, -1, -1, -1);
#pragma unroll
          for (int i = 0; i < MT; ++i)
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                a, xq[i], acc[j][i], 4, 4, 0, (int)e[j], 0, (int)xe[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float sc = mx_scale(e[j]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const u32x4 a = mx_word<DT>(W[d][j][q], sc);
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[j][i] = T::mfma(a, X[d][i][q], acc[j][i]);
          }
        }
      }
      load(d, s + d + D);
    }
  }
  __syncthreads();
  f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[(wave * NT * MT + j * MT + i) * 64 + lane] = acc[j][i];
  __syncthreads();
  for (int o = t; o < NT * MT * 64; o += NTHR) {
    f32x4 v = red[o];
#pragma unroll
    for (int k = 1; k < KW; ++k) v += red[k * NT * MT * 64 + o];
    const int tile = o >> 6;
    put(tile / MT, tile % MT, o & 63, v);
  }
}

// Four consecutive columns of a row; vec: N and out allow 8-byte stores.
template <int DT>
__device__ __forceinline__ void mx_store4(uint16_t* row, int n, int N, bool vec, const f32x4& v) {
  if (vec) {
    if (n < N)
      *reinterpret_cast<u32x2*>(row + n) =
          (u32x2){T16<DT>::pack2(v[0], v[1]), T16<DT>::pack2(v[2], v[3])};
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (n + q < N) row[n + q] = T16<DT>::round1(v[q]);
}

template <int DT, bool QQ, int MT, int NT, int KW>
__global__ __launch_bounds__(64 * KW) void mx_skinny_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ w,
    const uint8_t* __restrict__ scales, uint16_t* __restrict__ out, int M, int N, int G) {
  extern __shared__ __align__(16) unsigned char lds[];
  const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * (16 * MT);
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int64_t xb = (int64_t)G * 64;           // bytes per x row
  const unsigned char* xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i + r;
    xp[i] = reinterpret_cast<const unsigned char*>(x) + (m < M ? m : m0) * xb + 64 * c;
  }
  const bool vec = N % 4 == 0 && (uintptr_t)out % 8 == 0;
  mx_skinny_tile<DT, QQ, MT, NT, KW>(
      xp, w + (int64_t)n0 * G * 4, scales + (int64_t)n0 * G, min(16 * NT, N - n0), G, lds,
      [&](int j, int i, int l, const f32x4& v) {
        const int m = m0 + 16 * i + (l & 15);
        if (m < M) mx_store4<DT>(out + (int64_t)m * N, n0 + 16 * j + 4 * (l >> 4), N, vec, v);
      });
}

// gather_qmm: a workgroup's 16 MT rows are up to R = 16 MT / Mi pairs of one
// expert, found in the workgroup (FUSED: P <= 256; blockIdx.y is a pair, the
// first of every R pairs of an expert in pair order does their work) or in the
// prep kernels' tables.  Pairs whose expert or x batch does not exist get zeros.
template <int DT, int MT, int NT, int KW, bool FUSED>
__global__ __launch_bounds__(64 * KW) void mx_gather_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ w,
    const uint8_t* __restrict__ scales, const int32_t* __restrict__ lhs,
    const int32_t* __restrict__ rhs, uint16_t* __restrict__ out, const int32_t* __restrict__ ws,
    int P, int B, int Mi, int N, int G, int E) {
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ int s_pair[16 * MT];
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int R = 16 * MT / Mi;
  int n0, e, len;
  if constexpr (FUSED) {
    __shared__ uint64_t s_match[KW];
    const int p = blockIdx.y;
    auto expert = [&](int q) {
      const int k = rhs[q], b = x_batch(lhs, q, P, B);
      return k >= 0 && k < E && b >= 0 && b < B ? k : E;
    };
    e = __builtin_amdgcn_readfirstlane(expert(p));
    const bool match = t < P && expert(t) == e;
    const uint64_t m = __ballot(match);
    if (lane == 0) s_match[t >> 6] = m;
    __syncthreads();
    int before = 0, all = 0, mine = 0;          // of e's pairs: before p, in all, before t
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const uint64_t v = s_match[k];
      const int lo = p - 64 * k, lt = t - 64 * k;
      all += __popcll(v);
      before += __popcll(lo >= 64 ? v : lo <= 0 ? 0 : v & ((1ull << lo) - 1));
      mine += __popcll(lt >= 64 ? v : lt <= 0 ? 0 : v & ((1ull << lt) - 1));
    }
    if (before % R) return;                     // uniform
    len = min(R, all - before);
    if (match && mine >= before && mine < before + len) s_pair[mine - before] = t;
    n0 = blockIdx.x * (16 * NT);
  } else {
    int seg, col;
    const int ncol = (N + 16 * NT - 1) / (16 * NT);
    if (!grouped_tile(blockIdx.x, ws[0], ncol, seg, col)) return;
    const int32_t* perm = ws + 1;
    const int st0 = perm[P + seg];
    len = perm[2 * P + seg];
    e = __builtin_amdgcn_readfirstlane(perm[3 * P + seg]);
    if (t < len) s_pair[t] = perm[st0 + t];
    n0 = col * (16 * NT);
  }
  __syncthreads();
  const int rows = len * Mi, nrows = min(16 * NT, N - n0);
  if (e >= E) {
    for (int i = t; i < rows * nrows; i += 64 * KW) {
      const int a = i / nrows, q = a / Mi;
      out[((int64_t)s_pair[q] * Mi + a - q * Mi) * N + n0 + i - a * nrows] = 0;
    }
    return;
  }
  const int64_t xb = (int64_t)G * 64;
  const unsigned char* xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int a = 16 * i + r < rows ? 16 * i + r : 0, q = a / Mi;
    xp[i] = reinterpret_cast<const unsigned char*>(x) +
            ((int64_t)x_batch(lhs, s_pair[q], P, B) * Mi + a - q * Mi) * xb + 64 * c;
  }
  const int64_t row0 = (int64_t)e * N + n0;
  const bool vec = N % 4 == 0 && (uintptr_t)out % 8 == 0;
  mx_skinny_tile<DT, false, MT, NT, KW>(
      xp, w + row0 * G * 4, scales + row0 * G, nrows, G, lds,
      [&](int j, int i, int l, const f32x4& v) {
        const int a = 16 * i + (l & 15), q = a / Mi;
        if (a < rows)
          mx_store4<DT>(out + ((int64_t)s_pair[q] * Mi + a - q * Mi) * N,
                        n0 + 16 * j + 4 * (l >> 4), N, vec, v);
      });
}

// ---- host side ---------------------------------------------------------------

// Largest dynamic LDS of a workgroup here, and so the largest K: 16 NT rows of
// scales have to fit.
constexpr int64_t kMxLdsMax = 156 * 1024;

// K waves: a function of N and K alone.
inline int mx_kw(int64_t N) { return (N + 15) / 16 < 640 ? 8 : 4; }

template <int DT, bool QQ>
int MxSkinnyLaunch<DT, QQ>::run(const void* x, const uint32_t* w, const uint8_t* s, void* out,
                                int64_t M, int64_t N, int64_t K, hipStream_t st, int* nlaunch) {
  const int64_t G = K / kMxGroup;
  auto go = [&](auto mt, auto nt, auto kw) -> int {
    constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value, KW = decltype(kw)::value;
    const size_t lds = mx_skinny_lds<MT, NT, KW>(G);
    const int64_t gx = (N + 16 * NT - 1) / (16 * NT), gy = (M + 16 * MT - 1) / (16 * MT);
    if ((int64_t)lds > kMxLdsMax || gy > 65535) return kStatusUnsupported;
    const auto kern = &mx_skinny_kernel<DT, QQ, MT, NT, KW>;
    static std::atomic<uint64_t> lds_set{0};
    if (hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(kern), (int)kMxLdsMax,
                                        lds_set))
      return (int)e;
    hipLaunchKernelGGL(kern, dim3((unsigned)gx, (unsigned)gy), dim3(64 * KW), lds, st,
                       (const uint16_t*)x, w, s, (uint16_t*)out, (int)M, (int)N, (int)G);
    *nlaunch += 1;
    return 0;
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I4 = std::integral_constant<int, 4>;
  using I8 = std::integral_constant<int, 8>;
  if (mx_kw(N) == 8) {
    if (M <= 16) return go(I1{}, I1{}, I8{});
    if (M <= 32) return go(I2{}, I2{}, I8{});
    return go(I4{}, I2{}, I8{});
  }
  if (M <= 16) return go(I1{}, I2{}, I4{});
  if (M <= 32) return go(I2{}, I2{}, I4{});
  return go(I4{}, I2{}, I4{});
}

template <int DT>
int MxGatherLaunch<DT>::run(const void* x, const uint32_t* w, const uint8_t* s,
                            const int32_t* lhs, const int32_t* rhs, void* out, int64_t P,
                            int64_t B, int64_t M, int64_t N, int64_t K, int64_t E, void* ws,
                            hipStream_t st, int* nlaunch) {
  const int64_t G = K / kMxGroup;
  auto go = [&](auto mt, auto nt, auto fused) -> int {
    constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value, KW = 4;
    constexpr bool FUSED = decltype(fused)::value;
    const size_t lds = mx_skinny_lds<MT, NT, KW>(G);
    const int64_t ncol = (N + 16 * NT - 1) / (16 * NT), R = 16 * MT / M;
    if ((int64_t)lds > kMxLdsMax) return kStatusUnsupported;
    dim3 grid((unsigned)ncol, (unsigned)P);
    if (!FUSED) {
      const int64_t nwg = (class_seg_bound(P, R, 0, E) * ncol + 7) / 8 * 8;
      if (nwg > INT32_MAX) return kStatusUnsupported;
      if (int rc = launch_prep(rhs, lhs, P, E, B, (int)R, ws, st)) return rc;
      *nlaunch += kPrepLaunches;
      grid = dim3((unsigned)nwg);
    }
    const auto kern = &mx_gather_kernel<DT, MT, NT, KW, FUSED>;
    static std::atomic<uint64_t> lds_set{0};
    if (hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(kern), (int)kMxLdsMax,
                                        lds_set))
      return (int)e;
    hipLaunchKernelGGL(kern, grid, dim3(64 * KW), lds, st, (const uint16_t*)x, w, s, lhs, rhs,
                       (uint16_t*)out, (const int32_t*)ws, (int)P, (int)B, (int)M, (int)N,
                       (int)G, (int)E);
    *nlaunch += 1;
    return 0;
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I4 = std::integral_constant<int, 4>;
  if (P <= kGatherFusedMaxP && P * M < kGroupedMinRows) return go(I1{}, I1{}, std::true_type{});
  return go(I4{}, I2{}, std::false_type{});
}

}  // namespace mq
