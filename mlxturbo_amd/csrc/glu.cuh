// The dense gated feed-forward block over affine codes: h = act(x . Wg^T) * (x .
// Wu^T), few rows of x (this file) and many (glu_wide.cuh).
//
// Sums in float over the dequantized T weights, act in float, one rounding to
// T; with gf and uf the two sums are written as well (float, for the gradient).
//
// One row runs qmv_quad.cuh's gated form.  Up to 16 rows, a workgroup of 16 waves, one
// per CU, runs up to 16 tiles of 8 output columns.  A tile's A operand of
// v_mfma_f32_16x16x32 is 8 rows of the gate matrix and the same 8 of the up
// matrix, so both sums of a column are in one accumulator.
//  * The x rows lie in LDS once for all tiles, and so do the tiles' scales and biases
//    (a dword per group), both in slices of K where they do not fit: no step loads
//    either.  Read per step, 16 bytes of 16 rows at a time, the scales alone cost 6.8 of
//    27.7 us (loads without the arithmetic; N=17408 K=5120, weights from memory).
//  * A tile's K range is cut into units of one 128-byte line of each row; the units of
//    all the workgroup's tiles, in order, are dealt to the waves in contiguous
//    runs that differ by one unit at most.  A wave streams its run one unit ahead,
//    without a stop at the tiles' ends: 16 waves hold 64 KB of loads in flight per CU; two,
//    three and four units ahead took 0.9, 1.9 and 2.9 us more of 28, as the scales then
//    wait behind the weights.  A run of at most one tile's units touches at most two
//    tiles, whose sums meet the other waves' in LDS at the end, added in wave order: an
//    order that depends on the call's sizes and the CU count alone.
//  * A load instruction reads one whole line of 8 rows of one matrix, non-temporal: lane
//    (r = lane & 15, c = lane >> 4) the 16-byte chunk 2 c + (r >> 3) of row r & 7.  The
//    operand wants rows 8 .. 15 to be the up matrix's: lanes r < 8 and r >= 8 of a
//    gate and an up register change places by one DPP move each, after which both hold
//    chunk 2 c, or 2 c + 1, of 16 rows.
// Bound by the exact dequantization (VALU issue 73% of the CUs' busy time; 20 VALU per 8 codes; v_fma_mix, v_cvt_pk and DPP moves
// issue every 4.9 cycles, and and shift every 2.8) over the 15 us after the scales, whose
// read and barrier take 5.5, and by the last workgroups' 9 tiles against 8.5 on average:
// N=17408 K=5120, 4 bits, 25.9, 26.6 and 34.3 us for 2, 8 and 16 rows (100 MB: 20 us at the
// rate of a copy); 8 bits 36.7, 37.4 and 44.7; N=4096 K=4096 11.4, 12.3 and 13.3.
#pragma once
#include "glu_act.cuh"
#include "stream_tile.cuh"

namespace mq {

constexpr int kGluWaves = 16;
constexpr int kGluTiles = 16;                   // most tiles of a workgroup
constexpr int kGluCols = 8;                     // output columns of a tile

template <int BITS>
struct GluGeom {
  static constexpr int PC = 128 / BITS;         // codes per 16-byte chunk
  static constexpr int UC = 8 * PC;             // codes per row and unit
};

// LDS: the waves' two sums (in place of x and scales, at the end), then the tiles' sums
// where K is sliced.
constexpr int kGluPart = kGluWaves * 2 * 1024;
constexpr int kGluSum = kGluTiles * 1024;

// Bytes between x rows of a slice of `codes` codes: an odd number of 16-byte
// chunks, so that a fragment's 16 rows lie in distinct banks.
__host__ __device__ inline int glu_xstride(int codes) { return (codes * 2 + 31) / 32 * 32 + 16; }
// Dwords between rows' scales of a slice: an odd multiple of 4, so that 16 rows' and 4
// groups' lie in distinct banks.
__host__ __device__ inline int glu_sstride(int groups) { return (groups + 3) / 8 * 8 + 4; }

// LDS of a slice of `units` units: x of M rows, scales of `tiles` tiles.
template <int BITS, int GS>
__host__ __device__ inline size_t glu_slice_bytes(int64_t M, int tiles, int units) {
  constexpr int UC = GluGeom<BITS>::UC;
  const size_t n = (size_t)M * glu_xstride(units * UC) +
                   (size_t)tiles * 2 * kGluCols * 4 * glu_sstride(units * (UC / GS));
  return ((n > (size_t)kGluPart ? n : (size_t)kGluPart) + 15) & ~(size_t)15;
}

// A lane's weight row in a tile whose first is row n0 (the last one, past N), and its byte of
// unit s in a row of rowB: chunks past the row read its last one.
__host__ __device__ inline int glu_lane_row(int lane, int64_t n0, int N) {
  const int last = (int)(N - 1 - n0), r = lane & 7;
  return r < last ? r : last;
}
__host__ __device__ inline uint32_t glu_lane_byte(int lane, int s, uint32_t rowB) {
  const uint32_t o = 128u * (uint32_t)s + 16u * (2 * (lane >> 4) + ((lane & 15) >> 3));
  return o < rowB - 16u ? o : rowB - 16u;
}
// Its piece of P groups from group g on of a row's G: past them, the last (and zeros count).
__host__ __device__ inline int glu_piece_at(int g, int G, int P) { return g < G - P ? g : G - P; }

// Lanes 8 .. 15 of every 16 of a from lanes 0 .. 7 of b (HIGH), or the reverse.
template <bool HIGH>
__device__ __forceinline__ uint32_t swap_halves(uint32_t a, uint32_t b) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, 0x128, 0xf, HIGH ? 0xc : 0x3, false);
}

template <int DT, int BITS, int GS>
__global__ __launch_bounds__(64 * kGluWaves) void glu_skinny_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ wg,
    const uint16_t* __restrict__ sg, const uint16_t* __restrict__ bg,
    const uint32_t* __restrict__ wu, const uint16_t* __restrict__ su,
    const uint16_t* __restrict__ bu, uint16_t* __restrict__ out, float* __restrict__ gf,
    float* __restrict__ uf, int M, int N, int K, int act, int tiles, int slice) {
  using T = T16<DT>;
  constexpr int UC = GluGeom<BITS>::UC, PC = GluGeom<BITS>::PC;
  constexpr int GU = UC / GS;                   // groups per unit
  constexpr int WP = BITS == 4 ? 4 : 2;         // MFMAs per chunk
  constexpr int R = 2;                          // units in registers
  extern __shared__ __align__(16) unsigned char lds[];
  f32x4* part = reinterpret_cast<f32x4*>(lds);
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int t0 = (int)((int64_t)tiles * blockIdx.x / gridDim.x);
  const int nt = (int)((int64_t)tiles * (blockIdx.x + 1) / gridDim.x) - t0;
  const int S = (K + UC - 1) / UC;              // units of a row
  const int G = K / GS;
  const uint32_t rowB = (uint32_t)K * BITS / 8;
  const int xs = glu_xstride(slice * UC), ss = glu_sstride(slice * GU);
  unsigned char* xl = lds;
  uint32_t* sl = reinterpret_cast<uint32_t*>(lds + M * xs);
  f32x4* sums = reinterpret_cast<f32x4*>(
      lds + glu_slice_bytes<BITS, GS>(M, (tiles + (int)gridDim.x - 1) / (int)gridDim.x, slice));

  u32x4 W[R][2];                                // a line of the gate's rows, and of the up's
  const unsigned char *pg = nullptr, *pu = nullptr;
  uint32_t ro = 0;
  // tile j's first row in both matrices, and this lane's row (the last, past N)
  auto tile_at = [&](int j) {
    const int64_t n0 = (int64_t)(t0 + j) * kGluCols;
    pg = reinterpret_cast<const unsigned char*>(wg) + n0 * rowB;
    pu = reinterpret_cast<const unsigned char*>(wu) + n0 * rowB;
    ro = (uint32_t)glu_lane_row(lane, n0, N) * rowB;
  };
  // unit s of that tile into slot b
  auto load = [&](auto bc, int s) {
    constexpr int b = decltype(bc)::value;
    const uint32_t o = ro + glu_lane_byte(lane, s, rowB);
    W[b][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(pg + o));
    W[b][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(pu + o));
  };

  for (int s0 = 0; s0 < S; s0 += slice) {
    const int ns = min(slice, S - s0);
    const int units = nt * ns;
    const int i0 = units * wave / kGluWaves, i1 = units * (wave + 1) / kGluWaves;
    int j = i0 / ns, s = i0 - j * ns;           // the unit computed
    int jl = j, sl_ = s;                        // and the one loaded next
    // the next load, which stays at the run's last unit
    auto advance = [&](int i) {
      if (i + 1 < i1) {
        if (++sl_ == ns) {
          sl_ = 0;
          tile_at(++jl);
        }
      }
    };
    // The slice's scales and biases, gate rows, then up rows, in pieces of P groups, and x:
    // the first SB and XB pieces of each thread are read ahead of the weights.  Reads past the
    // slice's pieces are of the last rows again, those past K leave zeros.
    bool big = false;
    const int rows = nt * kGluCols, g0 = s0 * GU, ng = ns * GU;
    const int k0 = s0 * UC, ch = ns * UC / 8;   // 16-byte chunks of a row of x
    auto x_at = [&](int i) {
      const int m = i / ch, k = k0 + 8 * (i - m * ch);
      const u32x4 v =
          *reinterpret_cast<const u32x4*>(x + (int64_t)min(m, M - 1) * K + min(k, K - 8));
      return k < K ? v : (u32x4){0, 0, 0, 0};
    };
    auto x_put = [&](int i, u32x4 v) {
      const int m = i / ch;
      if (i < M * ch) *reinterpret_cast<u32x4*>(xl + m * xs + 16 * (i - m * ch)) = v;
    };
    auto start = [&] {
      tile_at(jl);
      load(std::integral_constant<int, 0>{}, s0 + sl_);
      advance(i0);
      if (s0) __syncthreads();                  // the last slice's sums are read
    };
    auto fill = [&](auto pc) {
      constexpr int P = decltype(pc)::value, SB = 2, XB = 2, TH = 64 * kGluWaves;
      using V = std::conditional_t<P == 8, u32x4, uint16_t>;
      const int per = ng / P, n = 2 * rows * per;
      struct Piece { V s, b; };
      auto at = [&](int i) {
        const int q = i / per, g = g0 + (i - q * per) * P;
        const bool up = q >= rows;
        const int64_t o =
            (int64_t)min(t0 * kGluCols + (up ? q - rows : q), N - 1) * G + glu_piece_at(g, G, P);
        Piece v;
        v.s = *reinterpret_cast<const V*>((up ? su : sg) + o);
        v.b = *reinterpret_cast<const V*>((up ? bu : bg) + o);
        return g < G ? v : Piece{};
      };
      auto put = [&](int i, const Piece& v) {
        if (i >= n) return;
        const int q = i / per;
        const bool up = q >= rows;
        const int k = up ? q - rows : q;
        // row k of its matrix is row k % 8, or 8 + k % 8, of tile k / 8
        uint32_t* d = sl + ((k >> 3) * 16 + (up ? 8 : 0) + (k & 7)) * ss + (i - q * per) * P;
        if constexpr (P == 8) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t s2 = v.s[2 * h + e], b2 = v.b[2 * h + e];
              o[2 * e] = (s2 & 0xffffu) | b2 << 16;
              o[2 * e + 1] = s2 >> 16 | (b2 & 0xffff0000u);
              big |= needs_plain(T::to_f32((uint16_t)s2));
              big |= needs_plain(T::to_f32((uint16_t)(s2 >> 16)));
            }
            *reinterpret_cast<u32x4*>(d + 4 * h) = o;
          }
        } else {
          *d = v.s | (uint32_t)v.b << 16;
          big |= needs_plain(T::to_f32(v.s));
        }
      };
      Piece sv[SB];
      u32x4 xv[XB];
#pragma unroll
      for (int u = 0; u < SB; ++u) sv[u] = at(t + u * TH);
#pragma unroll
      for (int u = 0; u < XB; ++u) xv[u] = x_at(t + u * TH);
      start();
#pragma unroll
      for (int u = 0; u < SB; ++u) put(t + u * TH, sv[u]);
#pragma unroll
      for (int u = 0; u < XB; ++u) x_put(t + u * TH, xv[u]);
#pragma unroll 4
      for (int i = t + SB * TH; i < n; i += TH) put(i, at(i));
    };
    if (G % 8 == 0 && g0 % 8 == 0 && ng % 8 == 0 &&
        (((uintptr_t)sg | (uintptr_t)bg | (uintptr_t)su | (uintptr_t)bu) & 15u) == 0)
      fill(std::integral_constant<int, 8>{});
    else
      fill(std::integral_constant<int, 1>{});
#pragma unroll 4
    for (int i = t + 2 * 64 * kGluWaves; i < M * ch; i += 64 * kGluWaves) x_put(i, x_at(i));
    const bool plain = __syncthreads_or(big);
    // rows past M repeat the last one: their columns are not stored
    const unsigned char* xu = xl + min(r, M - 1) * xs + 4 * PC * c + s * (2 * UC);
    const uint32_t* sr = sl + (j * 16 + r) * ss + s * GU;
    const int xwrap = ns * 2 * UC, swrap = 16 * ss - ns * GU;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f}, head = acc;
    const int j0 = j;
    // A SIMD's waves take turns by their progress: issued oldest first, the first ended
    // 13 us before the last, which then waited for memory alone (28.1 against 26.6 us).
    const int p1 = i0 + (i1 - i0) / 4, p2 = i0 + (i1 - i0) / 2, p3 = p2 + (i1 - i0) / 4;
    auto prio = [&](int i) {
      if (i < p1) __builtin_amdgcn_s_setprio(3);
      else if (i < p2) __builtin_amdgcn_s_setprio(2);
      else if (i < p3) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
    };
    auto step = [&](auto bc, auto plainc, int i) {
      constexpr int b = decltype(bc)::value;
      constexpr bool PLAIN = decltype(plainc)::value;
      load(std::integral_constant<int, (b + R - 1) % R>{}, s0 + sl_);
      advance(i + R - 1);
#pragma unroll
      for (int u = 0; u < 2; ++u) {             // codes (2 c + u) PC .. of the unit
        const uint32_t sb = sr[(2 * c + u) * PC / GS];
        const GroupScale g = make_group(T::to_f32((uint16_t)sb), T::to_f32((uint16_t)(sb >> 16)));
        uint32_t w[4], o[WP][4];
#pragma unroll
        for (int d = 0; d < 4; ++d)
          w[d] = u ? swap_halves<false>(W[b][1][d], W[b][0][d])
                   : swap_halves<true>(W[b][0][d], W[b][1][d]);
#pragma unroll
        for (int q = 0; q < WP; ++q) {
          if constexpr (BITS == 4) {
            if constexpr (PLAIN) deq_word_plain<DT, 4>(w[q], g, o[q]);
            else deq4_word<DT>(w[q], g, o[q]);
          } else {
            if constexpr (PLAIN) {
              deq_word_plain<DT, 8>(w[2 * q], g, o[q]);
              deq_word_plain<DT, 8>(w[2 * q + 1], g, o[q] + 2);
            } else {
              deq8_word<DT>(w[2 * q], g, o[q]);
              deq8_word<DT>(w[2 * q + 1], g, o[q] + 2);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < WP; ++q) {
          const u32x4 xv = *reinterpret_cast<const u32x4*>(xu + 2 * (PC * u + 8 * q));
          acc = T::mfma((u32x4){o[q][0], o[q][1], o[q][2], o[q][3]}, xv, acc);
        }
      }
      xu += 2 * UC;
      sr += GU;
      if (++s == ns) {                          // the next tile
        s = 0;
        ++j;
        xu -= xwrap;
        sr += swrap;
        if (i + 1 < i1) {
          head = acc;
          acc = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
      }
    };
    auto run = [&](auto plainc) {
      int i = i0;
      for (; i + R <= i1; i += R) {
        prio(i);
        step(std::integral_constant<int, 0>{}, plainc, i);
        step(std::integral_constant<int, 1>{}, plainc, i + 1);
      }
      if (i < i1) step(std::integral_constant<int, 0>{}, plainc, i);
    };
    if (__builtin_expect(!plain, 1)) run(std::false_type{});
    else run(std::true_type{});
    // the run's last tile's sum is in acc, that of the tile before it, if there is one, in head
    const bool two = i0 < i1 && (i1 - 1) / ns > j0;
    __syncthreads();                            // x and the scales are read
    part[wave * 128 + lane] = two ? head : acc;
    if (two) part[wave * 128 + 64 + lane] = acc;
    __syncthreads();
    // wave w: tile w's sums, in the order of the runs
    if (wave < nt) {
      const int u0 = wave * ns, u1 = u0 + ns;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (s0) v = sums[wave * 64 + lane];
      for (int w = 0; w < kGluWaves; ++w) {
        const int a0 = units * w / kGluWaves, a1 = units * (w + 1) / kGluWaves;
        if (a0 < u1 && a1 > u0 && a0 < a1) v += part[(w * 2 + wave - a0 / ns) * 64 + lane];
      }
      if (s0 + ns < S) {
        sums[wave * 64 + lane] = v;
      } else {
        // rows 4 c .. + 3 of the tile: gate columns in c < 2, up columns in c >= 2
        f32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __shfl_xor(v[e], 32);
        if (c < 2 && r < M) {
          const int n = (t0 + wave) * kGluCols + 4 * c;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (n + e < N) {
              out[(int64_t)r * N + n + e] = T::round1(glu_act(v[e], act) * o[e]);
              if (gf) {
                gf[(int64_t)r * N + n + e] = v[e];
                uf[(int64_t)r * N + n + e] = o[e];
              }
            }
          }
        }
      }
    }
  }
}

// Most LDS of a workgroup.
constexpr int kGluLdsMax = 160 * 1024 - 1024;

// Workgroups of a launch: one per CU, more where that would be over 16 tiles each; and x and
// scales in equal slices of whole units, as the LDS of `rows` rows needs.
struct GluSlices {
  int64_t wgs, units;
  size_t lds;
};
template <int BITS, int GS>
inline GluSlices glu_slices(int64_t rows, int64_t tiles, int64_t S, int cus) {
  const int64_t per = (tiles + (int64_t)cus * kGluTiles - 1) / ((int64_t)cus * kGluTiles);
  GluSlices p{tiles < cus * per ? tiles : cus * per, S, 0};
  const int most = (int)((tiles + p.wgs - 1) / p.wgs);
  for (int64_t n = 1;; ++n) {
    p.units = (S + n - 1) / n;
    p.lds = glu_slice_bytes<BITS, GS>(rows, most, (int)p.units) + (p.units < S ? kGluSum : 0);
    if (p.lds <= (size_t)kGluLdsMax) return p;
  }
}

template <int DT, int BITS, int GS>
int GluSkinnyLaunch<DT, BITS, GS>::run(const GluArgs& a, int64_t m0, int64_t M, int64_t rows,
                                       hipStream_t st) {
  constexpr int UC = GluGeom<BITS>::UC;
  const int64_t tiles = (a.N + kGluCols - 1) / kGluCols, S = (a.K + UC - 1) / UC;
  const GluSlices p = glu_slices<BITS, GS>(rows, tiles, S, device_cu_count());
  const auto kern = &glu_skinny_kernel<DT, BITS, GS>;
  static std::atomic<uint64_t> lds_set{0};
  if (hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(kern), kGluLdsMax, lds_set))
    return (int)e;
  const int64_t o = m0 * a.N;
  hipLaunchKernelGGL(kern, dim3((unsigned)p.wgs), dim3(64 * kGluWaves), p.lds, st,
                     (const uint16_t*)a.x + m0 * a.K, a.wg, (const uint16_t*)a.sg,
                     (const uint16_t*)a.bg, a.wu, (const uint16_t*)a.su, (const uint16_t*)a.bu,
                     (uint16_t*)a.out + o, a.gf ? a.gf + o : nullptr, a.uf ? a.uf + o : nullptr,
                     (int)M, (int)a.N, (int)a.K, a.act, (int)tiles, (int)p.units);
  return 0;
}

}  // namespace mq
