// The dense gated feed-forward block over affine codes: h = act(x . Wg^T) * (x .
// Wu^T), few rows of x (this file) and many (glu_wide.cuh).
//
// Sums in float over the dequantized T weights, act in float, one rounding to
// T; with gf and uf the two sums are written as well (float, for the gradient).
//
// Up to 16 rows the weight stream bounds the call.  A workgroup of 16 waves, one
// per CU, runs up to 16 tiles of 8 output columns.  A tile's A operand of
// v_mfma_f32_16x16x32 is 8 rows of the gate matrix and the same 8 of the up
// matrix, so both sums of a column are in one accumulator.
//  * The x rows lie in LDS once for all tiles (in slices of K where they do not
//    fit), so no step loads x.
//  * A tile's K range is cut into units of 256 bytes of each row; the units of
//    all the workgroup's tiles, in order, are dealt to the waves in contiguous
//    runs that differ by one unit at most.  A wave streams its run without a
//    stop at the tiles' ends; a run of at most one tile's units touches at
//    most two tiles, whose sums go to two places of LDS, and one wave per
//    tile adds them in wave order.  The order depends on N, K and the CU count
//    alone.
//  * Lane (r = lane & 15, c = lane >> 4) takes of row r's unit the 16-byte
//    pieces at 64 p + 16 c, p = 0..3: a load instruction reads whole 64-byte
//    sectors, the four of them whole lines.
#pragma once
#include "glu_launch.h"
#include "stream_tile.cuh"

namespace mq {

// act(g), in float.
__device__ __forceinline__ float glu_act(float g, int act) {
  // the tanh form 0.5 g (1 + tanh(z / 2)) is g / (1 + exp(-z))
  const float z = act == kActSilu ? g : kGeluZ * (g + kGeluCubic * g * g * g);
  return g / (1.0f + expf(-z));
}

constexpr int kGluWaves = 16;
constexpr int kGluTiles = 16;                   // most tiles of a workgroup
constexpr int kGluCols = 8;                     // output columns of a tile

template <int BITS>
struct GluGeom {
  static constexpr int UC = 2048 / BITS;        // codes per row and unit
  static constexpr int PC = 128 / BITS;         // codes per 16-byte piece
};

// LDS: the waves' two sums, the tiles' sums (K slices), x rows.
constexpr int kGluPart = kGluWaves * 2 * 1024;
constexpr int kGluSum = kGluTiles * 1024;

// Bytes between x rows of a slice of `codes` codes: an odd number of 16-byte
// chunks, so that a fragment's 16 rows lie in distinct banks.
__host__ __device__ inline int glu_xstride(int codes) { return (codes * 2 + 31) / 32 * 32 + 16; }

// SV: a unit's scales are read as dwords (whole units of K, 4-byte aligned scales
// and biases), else one by one.
template <int DT, int BITS, int GS, bool SV>
__global__ __launch_bounds__(64 * kGluWaves) void glu_skinny_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ wg,
    const uint16_t* __restrict__ sg, const uint16_t* __restrict__ bg,
    const uint32_t* __restrict__ wu, const uint16_t* __restrict__ su,
    const uint16_t* __restrict__ bu, uint16_t* __restrict__ out, float* __restrict__ gf,
    float* __restrict__ uf, int M, int N, int K, int act, int tiles, int slice) {
  using T = T16<DT>;
  constexpr int UC = GluGeom<BITS>::UC, PC = GluGeom<BITS>::PC;
  constexpr int GU = UC / GS;                   // groups per unit
  constexpr int WP = BITS == 4 ? 4 : 2;         // MFMAs per piece
  constexpr int ND = GU / 2;                    // their dwords
  static_assert(GU >= 2, "whole dwords of scales");
  extern __shared__ __align__(16) unsigned char lds[];
  f32x4* part = reinterpret_cast<f32x4*>(lds);
  f32x4* sums = reinterpret_cast<f32x4*>(lds + kGluPart);
  unsigned char* xl = lds + kGluPart + (slice * UC < K ? kGluSum : 0);
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int t0 = (int)((int64_t)tiles * blockIdx.x / gridDim.x);
  const int nt = (int)((int64_t)tiles * (blockIdx.x + 1) / gridDim.x) - t0;
  const int S = (K + UC - 1) / UC;              // units of a row
  const int G = K / GS;
  const uint32_t rowB = (uint32_t)K * BITS / 8;
  // gate rows in lanes r < 8, up rows in the others
  const unsigned char* wb = reinterpret_cast<const unsigned char*>(r < 8 ? wg : wu);
  const uint16_t* sb = r < 8 ? sg : su;
  const uint16_t* bb = r < 8 ? bg : bu;

  u32x4 W[2][4];
  uint32_t sc[2][2][SV ? ND : 4];               // [ring][scale, bias]: SV dwords, else the pieces'
  // unit s of tile t0 + j into slot b
  auto load = [&](auto bc, int j, int s) {
    constexpr int b = decltype(bc)::value;
    const int row = min((t0 + j) * kGluCols + (r & 7), N - 1);
    const unsigned char* wr = wb + (int64_t)row * rowB;
    const uint16_t* sr = sb + (int64_t)row * G;
    const uint16_t* br = bb + (int64_t)row * G;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      uint32_t o = 256u * (uint32_t)s + 64u * p + 16u * c;
      if constexpr (!SV) o = o < rowB ? o : 0u;
      W[b][p] = *reinterpret_cast<const u32x4*>(wr + o);
    }
    if constexpr (SV) {
      const uint32_t* s32 = reinterpret_cast<const uint32_t*>(sr + s * GU);
      const uint32_t* b32 = reinterpret_cast<const uint32_t*>(br + s * GU);
#pragma unroll
      for (int q = 0; q < ND; ++q) {
        sc[b][0][q] = s32[q];
        sc[b][1][q] = b32[q];
      }
    } else {
      // a piece past the row: zero scale and bias, so zero weights
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int k = s * UC + p * 4 * PC + c * PC, g = k < K ? k / GS : 0;
        const uint32_t sv = sr[g], bv = br[g];
        sc[b][0][p] = k < K ? sv : 0u;
        sc[b][1][p] = k < K ? bv : 0u;
      }
    }
  };
  // scale (i = 0) or bias (1) of piece p as a float
  auto param = [&](int b, int i, int p) -> float {
    uint16_t v;
    if constexpr (!SV) {
      v = (uint16_t)sc[b][i][p];
    } else if constexpr (4 * PC / GS == 4) {    // group 4 p + c
      const uint32_t d = c & 2 ? sc[b][i][2 * p + 1] : sc[b][i][2 * p];
      v = (uint16_t)(c & 1 ? d >> 16 : d);
    } else if constexpr (4 * PC / GS == 2) {    // 2 p + (c >> 1)
      v = (uint16_t)(c & 2 ? sc[b][i][p] >> 16 : sc[b][i][p]);
    } else {
      constexpr int per = GS / (4 * PC);        // p / per
      const int g = p / per;
      v = (uint16_t)(sc[b][i][g >> 1] >> (16 * (g & 1)));
    }
    return T::to_f32(v);
  };

  const int xs = glu_xstride(slice * UC);
  for (int ph = 0, s0 = 0; s0 < S; ++ph, s0 += slice) {
    const int ns = min(slice, S - s0);
    const int units = nt * ns;
    const int i0 = units * wave / kGluWaves, i1 = units * (wave + 1) / kGluWaves;
    int j = i0 / ns, s = i0 - j * ns;
    const int j0 = j;
    if (i0 < i1) load(std::integral_constant<int, 0>{}, j, s0 + s);
    if (ph) __syncthreads();                    // the last slice's x and sums are read
    {
      const int k0 = s0 * UC, ch = ns * UC / 8; // 16-byte chunks of a row
      for (int i = t; i < M * ch; i += 64 * kGluWaves) {
        const int m = i / ch, q = i - m * ch, k = k0 + 8 * q;
        u32x4 v = {0, 0, 0, 0};
        if (k < K) v = *reinterpret_cast<const u32x4*>(x + (int64_t)m * K + k);
        *reinterpret_cast<u32x4*>(xl + m * xs + 16 * q) = v;
      }
    }
    __syncthreads();
    // rows past M repeat the last one: their columns are not stored
    const unsigned char* xf = xl + min(r, M - 1) * xs + 2 * PC * c;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto step = [&](auto bc, int i) {
      constexpr int b = decltype(bc)::value;
      int jn = j, sn = s + 1;
      if (sn == ns) {
        sn = 0;
        ++jn;
      }
      const bool more = i + 1 < i1;
      load(std::integral_constant<int, b ^ 1>{}, more ? jn : j, s0 + (more ? sn : s));
      float sv[4], bv[4];
      bool big = false;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        sv[p] = param(b, 0, p);
        bv[p] = param(b, 1, p);
        big |= needs_plain(sv[p]);
      }
      const unsigned char* xu = xf + s * (2 * UC);
      auto mma = [&](int p, int q, const uint32_t* o) {
        const u32x4 xv = *reinterpret_cast<const u32x4*>(xu + 2 * (4 * PC * p + 8 * q));
        acc = T::mfma((u32x4){o[0], o[1], o[2], o[3]}, xv, acc);
      };
      if (__builtin_expect(!__any(big), 1)) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const GroupScale g = make_group(sv[p], bv[p]);
#pragma unroll
          for (int q = 0; q < WP; ++q) {
            uint32_t o[4];
            if constexpr (BITS == 4) {
              deq4_word<DT>(W[b][p][q], g, o);
            } else {
              deq8_word<DT>(W[b][p][2 * q], g, o);
              deq8_word<DT>(W[b][p][2 * q + 1], g, o + 2);
            }
            mma(p, q, o);
          }
        }
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const GroupScale g = make_group(sv[p], bv[p]);
#pragma unroll
          for (int q = 0; q < WP; ++q) {
            uint32_t o[4];
            if constexpr (BITS == 4) {
              deq_word_plain<DT, 4>(W[b][p][q], g, o);
            } else {
              deq_word_plain<DT, 8>(W[b][p][2 * q], g, o);
              deq_word_plain<DT, 8>(W[b][p][2 * q + 1], g, o + 2);
            }
            mma(p, q, o);
          }
        }
      }
      if (!more || sn == 0) {                   // the run's or the tile's end
        part[(wave * 2 + j - j0) * 64 + lane] = acc;
        acc = (f32x4){0.f, 0.f, 0.f, 0.f};
      }
      j = jn;
      s = sn;
    };
    for (int i = i0; i < i1; i += 2) {
      step(std::integral_constant<int, 0>{}, i);
      if (i + 1 < i1) step(std::integral_constant<int, 1>{}, i + 1);
    }
    __syncthreads();
    // wave w: tile w's sums, in the order of the runs
    if (wave < nt) {
      const int u0 = wave * ns, u1 = u0 + ns;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (ph) v = sums[wave * 64 + lane];
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

// Most LDS of a workgroup that holds x rows of one slice.
constexpr int kGluLdsMax = 160 * 1024 - 1024;

template <int DT, int BITS, int GS>
int GluSkinnyLaunch<DT, BITS, GS>::run(const GluArgs& a, int64_t m0, int64_t M, hipStream_t st) {
  constexpr int UC = GluGeom<BITS>::UC;
  const int64_t tiles = (a.N + kGluCols - 1) / kGluCols, S = (a.K + UC - 1) / UC;
  const int cus = device_cu_count();
  // one workgroup per CU, more where that would be over 16 tiles each
  const int64_t per = (tiles + (int64_t)cus * kGluTiles - 1) / ((int64_t)cus * kGluTiles);
  const int64_t wgs = tiles < cus * per ? tiles : cus * per;
  // x in equal slices of whole units
  int64_t slice = S;
  size_t lds = 0;
  for (int64_t n = 1;; ++n) {
    slice = (S + n - 1) / n;
    lds = (size_t)kGluPart + (n > 1 ? kGluSum : 0) + (size_t)M * glu_xstride((int)(slice * UC));
    if (lds <= (size_t)kGluLdsMax) break;
  }
  const uintptr_t any = (uintptr_t)a.sg | (uintptr_t)a.bg | (uintptr_t)a.su | (uintptr_t)a.bu;
  const bool sv = a.K % UC == 0 && any % 4 == 0;    // a row's groups are whole dwords then
  auto go = [&](auto svc) -> int {
    const auto kern = &glu_skinny_kernel<DT, BITS, GS, decltype(svc)::value>;
    static std::atomic<uint64_t> lds_set{0};
    if (hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(kern), kGluLdsMax, lds_set))
      return (int)e;
    const int64_t o = m0 * a.N;
    hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(64 * kGluWaves), lds, st,
                       (const uint16_t*)a.x + m0 * a.K, a.wg, (const uint16_t*)a.sg,
                       (const uint16_t*)a.bg, a.wu, (const uint16_t*)a.su, (const uint16_t*)a.bu,
                       (uint16_t*)a.out + o, a.gf ? a.gf + o : nullptr, a.uf ? a.uf + o : nullptr,
                       (int)M, (int)a.N, (int)a.K, a.act, (int)tiles, (int)slice);
    return 0;
  };
  return sv ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace mq
