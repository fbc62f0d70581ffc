// Products of few x rows with MXFP4 weights: the weight stream bounds them.
//
// out[m, n] = sum over groups g of 32 codes of 2^(e[n, g] - 127) *
// (x[m, g] . code[n, g]), summed in float by MFMAs of 16x16x32 over the
// weights' T values (T(code * 2^(e - 127))), or, QQ, of 16x16x128 over the
// codes of both operands with their scale bytes.
//
// A wave owns 16 NT weight rows and every KW-th step of K; the KW waves of a
// workgroup add their sums through LDS in wave order.  A step is 256 codes,
// the eight groups of a whole 128-byte line of a weight row, and the even and
// the odd groups have sums of their own, added at the end.  Lane (r = lane & 15,
// c = lane >> 4) takes two 16-byte pieces of weights, each a group:
//
//  * F = 1, up to 16 rows of x: row r's groups 2 c and 2 c + 1, each times the x
//    of the same group of x row r.
//  * F = 2, up to 8 rows: group 2 c + (r >> 3) of weight rows (r & 7) and 8 +
//    (r & 7), both times the same group of x row r & 7.  The MFMAs' blocks of
//    weight rows and x rows with r >> 3 equal are sums of even or odd groups,
//    the other blocks are not used.  Half the x per weight, and whole lines per
//    weight load.
//
// MFMA j multiplies codes 8 j .. 8 j + 7 of every lane's group (the order of k
// is the same on both sides, so it does not matter).  Either way a row's sums
// are made in the same order, a function of N and K alone, so its result does
// not depend on how many rows the call has.
//
// A step ahead, weights go to registers and x to the wave's own LDS by the
// global loads' LDS form, in whole row pieces of 512 bytes with the 16-byte
// chunks permuted (xswz) so that fragment reads hit distinct banks; the
// fragments are read to registers before the next step's x replaces them.  The
// tile's scale bytes are one contiguous block, copied to LDS first.  N=17408
// K=5120, us at 8 rows, weights from memory: 16.7 (on another card 16.0; partly from
// the last-level cache 13.8), and as much at one row.  Fragments straight from
// memory, 16 bytes of 64 different pieces per load, cost as much as the weights
// (18.4; 12.0 without the loads of x); a second step in flight is slower (18.0), and
// so are contiguous K slices per wave (17.5: a workgroup's waves then read far apart)
// and 16 or 64 weight rows per wave (17.9, 18.7).
//
// Groups past K: zero codes (outside the buffer range), scale byte 0 and x from
// a block of zeros, so no 0 * inf arises.  Rows of x past M read row 0 of the
// tile; their columns are not stored.
#pragma once
#include "mx_common.cuh"
#include "mx_launch.h"

namespace mq {

__device__ __align__(64) static const unsigned char mx_zeros[64] = {};

// Rows of x of a tile.
template <int F> constexpr int mx_rows() { return F == 2 ? 8 : 16; }

// Where chunk p of a step's 32 chunks of x row i lies: p ^ xswz(i).  A fragment
// read takes, in each 16 lanes, one chunk of 16 rows (F = 1) or chunks p and p +
// 4 of 8 rows (F = 2).
template <int F>
__device__ __forceinline__ int xswz(int i) {
  return F == 1 ? i : (i & 3) | ((i >> 2) << 3);
}

// Dynamic LDS: scales of 16 NT rows, then the waves' x; later the waves' sums.
template <int NT> __host__ __device__ inline size_t mx_skinny_scales(int64_t G) {
  return ((size_t)(16 * NT) * (size_t)G + 16 + 15) & ~(size_t)15;
}
template <int F, int NT, int KW>
__host__ __device__ inline size_t mx_skinny_lds(int64_t G) {
  const size_t in = mx_skinny_scales<NT>(G) + (size_t)KW * mx_rows<F>() * 512;
  const size_t red = (size_t)KW * NT * (F == 2 ? 2 : 1) * 1024;
  return in > red ? in : red;
}

// xrow(i): the x row of tile row i < mx_rows.  w, scales: the tile's first row;
// nrows <= 16 NT of them exist.  put(n, m, v): v[q] = the sum of the tile's
// weight row n + q and x row m.
template <int DT, bool QQ, int F, int NT, int KW, class XRow, class Put>
__device__ __forceinline__ void mx_skinny_tile(XRow xrow, const uint32_t* __restrict__ w,
                                               const uint8_t* __restrict__ scales, int nrows,
                                               int G, unsigned char* __restrict__ lds, Put put) {
  constexpr int NX = F == 2 ? 1 : 2;            // groups of an x row per lane and step
  constexpr int XB = mx_rows<F>() * 512, NI = XB / 1024;   // x bytes and loads per step
  constexpr int NTHR = 64 * KW;
  using T = T16<DT>;
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int S = (G + 7) >> 3;                   // wave: steps wave, wave + KW, ...
  const auto rw = wide_rsrc(w, (int64_t)nrows * G * 16);
  uint32_t skew;
  const auto rs = mx_scale_rsrc(scales, (int64_t)nrows * G, skew);
  const uint32_t sbytes = (uint32_t)(nrows * G) + skew;
  unsigned char* xl = lds + mx_skinny_scales<NT>(G) + wave * XB;
  // piece u of tile j: its weight row, and its group of the step
  auto wrow = [&](int j, int u) { return 16 * j + (F == 2 ? 8 * u + (r & 7) : r); };
  auto grp = [&](int u) { return 2 * c + (F == 2 ? r >> 3 : u); };

  uint32_t wo[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 0; u < 2; ++u) wo[j][u] = (uint32_t)(wrow(j, u) * G + grp(u)) * 16u;
  // x load i: rows 2 i and 2 i + 1, lane's chunk of the row
  const unsigned char* xp[NI];
  int xg[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = 2 * i + (lane >> 5), p = (lane & 31) ^ xswz<F>(row);
    xp[i] = reinterpret_cast<const unsigned char*>(xrow(row)) + 16 * p;
    xg[i] = p >> 2;
  }
  u32x4 W[2][NT][2];
  auto xload = [&](int s) {
    const bool in = s < S;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const unsigned char* a = in && 8 * s + xg[i] < G ? xp[i] + 512 * (int64_t)s : mx_zeros;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)a,
                                       (lds_void*)(xl + 1024 * i), 16, 0, 0);
    }
  };
  auto wload = [&](int b, int s) {
    const bool in = s < S;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        W[b][j][u] = __builtin_amdgcn_raw_buffer_load_b128(
            rw, in && 8 * s + grp(u) < G ? wo[j][u] + 128u * (uint32_t)s : 0x80000000u, 0, 0);
  };
  // the first scale pieces go out before the weights
  u32x4 sv[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    sv[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (uint32_t)(i * NTHR + t) * 16u, 0, 0);
  xload(wave);
  wload(0, wave);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t o = (uint32_t)(i * NTHR + t) * 16u;
    if (o < sbytes) *reinterpret_cast<u32x4*>(lds + o) = sv[i];
  }
  for (uint32_t o = (uint32_t)(2 * NTHR + t) * 16u; o < sbytes; o += NTHR * 16u)
    *reinterpret_cast<u32x4*>(lds + o) = __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0);
  __syncthreads();

  f32x4 acc[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 0; u < 2; ++u) acc[j][u] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // rows past the tile's last read its scales
  uint32_t so[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 0; u < 2; ++u)
      so[j][u] = skew + (uint32_t)(min(wrow(j, u), nrows - 1) * G + grp(u));
  const int xr = F == 2 ? r & 7 : r;
  const unsigned char* xf = xl + xr * 512;

  for (int s = wave; s < S; s += 2 * KW) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      // this step's loads are in
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 15));
      asm volatile("" ::: "memory");
      u32x4 X[NX][4];
#pragma unroll
      for (int u = 0; u < NX; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          X[u][q] = *reinterpret_cast<const u32x4*>(
              xf + (((4 * grp(u) + q) ^ xswz<F>(xr)) << 4));
      uint32_t e[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool v = 8 * (s + b * KW) + grp(u) < G;
          const uint32_t y = lds[v ? so[j][u] + 8u * (uint32_t)(s + b * KW) : skew];
          e[j][u] = v ? y : 0u;
        }
      // the fragments are read: their place may be refilled
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
      asm volatile("" ::: "memory");
      xload(s + (b + 1) * KW);
      wload(b ^ 1, s + (b + 1) * KW);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (QQ) {
        i32x8 xq[NX];
        uint32_t xe[NX];
#pragma unroll
        for (int u = 0; u < NX; ++u) {
          uint32_t top = 0;
#pragma unroll
          for (int q = 0; q < 16; ++q) top = mx_max2(top, X[u][q >> 2][q & 3] & 0x7fff7fffu);
          xe[u] = mx_scale_byte<DT>(max(top & 0xffffu, top >> 16));
          const float xs = mx_scale(xe[u]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t cw = mx_code_word<DT>(X[u][q], xs);
            xq[u][q] = (int)(xe[u] == 255 ? 0u : cw);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const i32x8 a = __builtin_shufflevector(bitcast<i32x4>(W[b][j][u]),
                                                    bitcast<i32x4>(W[b][j][u]), 0, 1, 2, 3, -1, -1,
                                                    -1, -1);
            acc[j][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                a, xq[u % NX], acc[j][u], 4, 4, 0, (int)e[j][u], 0, (int)xe[u % NX]);
          }
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float sc = mx_scale(e[j][u]);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[j][u] = T::mfma(mx_word<DT>(W[b][j][u][q], sc), X[u % NX][q], acc[j][u]);
          }
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  __syncthreads();
  // per wave: F = 1 the even and odd sums added, F = 2 both pieces as they are
  constexpr int NR = F == 2 ? NT * 2 : NT;
  f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if constexpr (F == 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) red[(wave * NR + 2 * j + u) * 64 + lane] = acc[j][u];
    } else {
      red[(wave * NR + j) * 64 + lane] = acc[j][0] + acc[j][1];
    }
  }
  __syncthreads();
  if constexpr (F == 2) {
    // piece 2 j + u: weight rows 16 j + 8 u + 4 h .. + 3 and x row m in lanes 16
    // h + m (even groups) and 16 (h + 2) + 8 + m (odd)
    for (int o = t; o < NR * 16; o += NTHR) {
      const int p = o >> 4, h = (o >> 3) & 1, m = o & 7;
      const f32x4* a = red + p * 64 + 16 * h + m;
      f32x4 v = a[0] + a[40];
#pragma unroll
      for (int k = 1; k < KW; ++k) v += a[k * NR * 64] + a[k * NR * 64 + 40];
      put(8 * p + 4 * h, m, v);
    }
  } else {
    for (int o = t; o < NR * 64; o += NTHR) {
      f32x4 v = red[o];
#pragma unroll
      for (int k = 1; k < KW; ++k) v += red[k * NR * 64 + o];
      const int l = o & 63;
      put(16 * (o >> 6) + 4 * (l >> 4), l & 15, v);
    }
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

template <int DT, bool QQ, int F, int NT, int KW>
__global__ __launch_bounds__(64 * KW) void mx_skinny_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ w,
    const uint8_t* __restrict__ scales, uint16_t* __restrict__ out, int M, int N, int G) {
  extern __shared__ __align__(16) unsigned char lds[];
  const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * mx_rows<F>();
  const bool vec = N % 4 == 0 && (uintptr_t)out % 8 == 0;
  mx_skinny_tile<DT, QQ, F, NT, KW>(
      [&](int i) { return x + (int64_t)(m0 + i < M ? m0 + i : m0) * G * 32; },
      w + (int64_t)n0 * G * 4, scales + (int64_t)n0 * G, min(16 * NT, N - n0), G, lds,
      [&](int n, int m, const f32x4& v) {
        if (m0 + m < M) mx_store4<DT>(out + (int64_t)(m0 + m) * N, n0 + n, N, vec, v);
      });
}

// gather_qmm: a workgroup's rows (mx_rows) are up to R = rows / Mi pairs of one
// expert, found in the workgroup (FUSED: P <= 256; blockIdx.y is a pair, the
// first of every R pairs of an expert in pair order does their work) or in the
// prep kernels' tables.  Pairs whose expert or x batch does not exist get zeros.
template <int DT, int F, int NT, int KW, bool FUSED>
__global__ __launch_bounds__(64 * KW) void mx_gather_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ w,
    const uint8_t* __restrict__ scales, const int32_t* __restrict__ lhs,
    const int32_t* __restrict__ rhs, uint16_t* __restrict__ out, const int32_t* __restrict__ ws,
    int P, int B, int Mi, int N, int G, int E) {
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ int s_pair[mx_rows<F>()];
  const int t = threadIdx.x, lane = t & 63;
  const int R = mx_rows<F>() / Mi;
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
  const int64_t row0 = (int64_t)e * N + n0;
  const bool vec = N % 4 == 0 && (uintptr_t)out % 8 == 0;
  mx_skinny_tile<DT, false, F, NT, KW>(
      [&](int i) {
        const int a = i < rows ? i : 0, q = a / Mi;
        return x + ((int64_t)x_batch(lhs, s_pair[q], P, B) * Mi + a - q * Mi) * G * 32;
      },
      w + row0 * G * 4, scales + row0 * G, nrows, G, lds, [&](int n, int m, const f32x4& v) {
        if (m >= rows) return;
        const int q = m / Mi;
        mx_store4<DT>(out + ((int64_t)s_pair[q] * Mi + m - q * Mi) * N, n0 + n, N, vec, v);
      });
}

// ---- host side ---------------------------------------------------------------

// Largest dynamic LDS of a workgroup here, and so the largest K: 16 NT rows of
// scales have to fit.
constexpr int64_t kMxLdsMax = 156 * 1024;

// Waves that share K: a function of N alone.
inline int mx_kw(int64_t N) { return (N + 15) / 16 < 640 ? 8 : 4; }

template <int DT, bool QQ>
int MxSkinnyLaunch<DT, QQ>::run(const void* x, const uint32_t* w, const uint8_t* s, void* out,
                                int64_t M, int64_t N, int64_t K, hipStream_t st, int* nlaunch) {
  const int64_t G = K / kMxGroup;
  auto go = [&](auto f, auto nt, auto kw) -> int {
    constexpr int F = decltype(f)::value, NT = decltype(nt)::value, KW = decltype(kw)::value;
    constexpr int R = mx_rows<F>();
    const size_t lds = mx_skinny_lds<F, NT, KW>(G);
    const int64_t gx = (N + 16 * NT - 1) / (16 * NT), gy = (M + R - 1) / R;
    if ((int64_t)lds > kMxLdsMax || gy > 65535 || !mx_grid_ok(gx, 64 * KW)) return kStatusUnsupported;
    const auto kern = &mx_skinny_kernel<DT, QQ, F, NT, KW>;
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
  // weight rows per wave: 16 where long K would make 32 leave CUs idle (N=4096
  // K=4096, 8 rows: 5.4 against 6.1 us; N=5120 K=17408 21.3 against 18.5)
  const bool one = mx_kw(N) == 8 && K < 8192;
  if (M <= 8)
    return one ? go(I2{}, I1{}, I8{}) : mx_kw(N) == 8 ? go(I2{}, I2{}, I8{}) : go(I2{}, I2{}, I4{});
  return one ? go(I1{}, I1{}, I8{}) : mx_kw(N) == 8 ? go(I1{}, I2{}, I8{}) : go(I1{}, I2{}, I4{});
}

template <int DT>
int MxGatherLaunch<DT>::run(const void* x, const uint32_t* w, const uint8_t* s,
                            const int32_t* lhs, const int32_t* rhs, void* out, int64_t P,
                            int64_t B, int64_t M, int64_t N, int64_t K, int64_t E, void* ws,
                            hipStream_t st, int* nlaunch) {
  const int64_t G = K / kMxGroup;
  auto go = [&](auto f, auto nt, auto fused) -> int {
    constexpr int F = decltype(f)::value, NT = decltype(nt)::value, KW = 4;
    constexpr bool FUSED = decltype(fused)::value;
    const size_t lds = mx_skinny_lds<F, NT, KW>(G);
    const int64_t ncol = (N + 16 * NT - 1) / (16 * NT), R = mx_rows<F>() / M;
    if ((int64_t)lds > kMxLdsMax || !mx_grid_ok(ncol, 64 * KW)) return kStatusUnsupported;
    dim3 grid((unsigned)ncol, (unsigned)P);
    if (!FUSED) {
      const int64_t nwg = (class_seg_bound(P, R, 0, E) * ncol + 7) / 8 * 8;
      if (!mx_grid_ok(nwg, 64 * KW)) return kStatusUnsupported;
      if (int rc = launch_prep(rhs, lhs, P, E, B, (int)R, ws, st)) return rc;
      *nlaunch += kPrepLaunches;
      grid = dim3((unsigned)nwg);
    }
    const auto kern = &mx_gather_kernel<DT, F, NT, KW, FUSED>;
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
  if (P <= kGatherFusedMaxP && P * M < kGroupedMinRows) {
    if (M <= 8) return go(I2{}, I1{}, std::true_type{});
    return go(I1{}, I1{}, std::true_type{});
  }
  return go(I1{}, I2{}, std::false_type{});
}

}  // namespace mq
