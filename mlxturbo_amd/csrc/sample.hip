// A token from each row of logits: temperature, the k largest, the most probable of
// mass p, those no less probable than min_p of the most probable, and a given uniform
// number.
//
// With m the row's largest logit and T its temperature, word i has mass w_i = exp((l_i -
// m) / T), evaluated in double and held as the integer W_i = round(2^s w_i), s = 44
// (less where 2^18 words and more could overflow the sum).  Integers make every sum
// exact, so a result depends on no order of additions, atomics or chunks; what they
// leave out, 2^-45 of the largest mass per word, is far below a float uniform number's
// own steps.  Order is by value, then by index (the lower first).  Kept are
//   top_k: the first k words (k >= 1),
//   top_p: of those, the words before which the mass is less than p times their sum (p
//          < 1; always the first),
//   min_p: of those, the words with w_i >= min_p (always the first).
// The token is the first word, in index order, up to which the kept mass is more than
// u times the kept mass of the row.  T = 0 takes the first word.  NaN logits are
// left out, as -inf; a row with nothing else gives token -1, log probability -inf.
//
// One row of 248320 16-bit words is half a megabyte: latency bounds a few rows, so a
// row is spread over workgroups (chunks of its tiles, up to 1024 of 64 granules or
// more), and the passes are launches for all rows whatever their settings.  (us of the
// steps, 248320 bf16 words: one row with k and p 3.3, 5.3 and 10.5 for 3 and 4; 64 rows of
// mixed settings 10.3, at 3 TB/s of logits, 22.7, 18.7 and 16.4.  Of the 22.7, the double
// arithmetic of the 22 rows that need masses is about 8 by instruction count; CUs are busy for
// 60% of the launch, as the other rows' workgroups end at once.  In the last step 64 CUs have
// a row each.)
//   1 each tile's first word.  Where k tiles hold a word, the k-th largest of their
//     first words is no larger than the k-th largest word: a bound (step 2 finds it)
//     above which lie few more than k words;
//   2 masses.  Rows without k and p: each tile's kept mass.  Rows with p alone: masses
//     by bins of (m - l) / T, 2048 of 1/64.  Rows with more k than such tiles: counts
//     by the same bins;
//   3 rows with k or p: a list of the words among which the cut falls: from the bound
//     on; up to the bin that holds the k-th word; or those of the bin in which p is
//     reached, and each tile's mass in the bins before it;
//   4 rows with k: the list sorted, the cut by a scan of its masses, and the word that u
//     points at among the kept words in index order.  Others: the cut by the list's
//     masses, and the word in the tile that u points at.
// Few workgroups (512) run 3 and 4 as one launch: the row's last one to have listed
// goes on.  A list of more than 4096 words (many equal logits, k in the thousands)
// overflows: step 4 then selects by radix over the row.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mq_common.h"
#include "sample_launch.h"

namespace mq {

namespace {

constexpr int kBins = kSampleBins, kList = kSampleList;
constexpr float kBinsPerNat = 64.0f;            // bins cover 32 nats, past which masses are 0
constexpr int kThreads = 512;

typedef unsigned long long u64;

// One row's settings.
struct RowSet {
  float T, p, min_p, u;
  int k;                                        // 0: all
  bool greedy, by_k, by_p;
};

__device__ __forceinline__ RowSet row_set(const SampleArgs& a, int r) {
  RowSet s;
  s.T = a.temperature ? a.temperature[r] : a.temperature0;
  s.p = a.top_p ? a.top_p[r] : a.top_p0;
  s.min_p = a.min_p ? a.min_p[r] : a.min_p0;
  s.k = a.top_k ? a.top_k[r] : a.top_k0;
  s.u = a.u[r];
  s.greedy = !(s.T > 0.0f);
  if (s.p <= 0.0f) s.k = 1;                     // the first word alone
  if (s.k >= a.V || s.k < 0) s.k = 0;
  s.by_k = s.k > 0;
  s.by_p = s.p < 1.0f && s.p > 0.0f;
  return s;
}

template <int DT> struct Granule { static constexpr int E = DT == kF32 ? 4 : 8; };

// Where a row lies among 16-byte granules: granule g holds words g E - off ...
template <int DT>
struct RowView {
  static constexpr int E = Granule<DT>::E;
  static constexpr int kSize = DT == kF32 ? 4 : 2;
  const unsigned char* p;                       // the row, down to a granule
  int off, V, n;                                // n: granules

  __device__ __forceinline__ RowView(const SampleArgs& a, int r) {
    const unsigned char* row =
        static_cast<const unsigned char*>(a.logits) + (int64_t)r * a.row_stride * kSize;
    off = (int)((uintptr_t)row % 16) / kSize;
    p = row - off * kSize;
    V = (int)a.V;
    n = (off + V + E - 1) / E;
  }
  __device__ __forceinline__ int first(int g) const { return g * E - off; }
  // words of granule g as floats; -inf for NaN and for places outside the row, which are
  // not read
  __device__ __forceinline__ void load(int g, float (&v)[E]) const {
    const int i0 = first(g);
    uint32_t d[4];
    if (i0 >= 0 && i0 + E <= V) {
      const u32x4 q = *reinterpret_cast<const u32x4*>(p + (int64_t)g * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = q[j];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = value(d, e);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = -__builtin_inff();
        if (i0 + e >= 0 && i0 + e < V) {
          if constexpr (DT == kF32) {
            v[e] = *reinterpret_cast<const float*>(p + (int64_t)g * 16 + 4 * e);
          } else {
            v[e] = T16<DT == kF32 ? kBF16 : DT>::to_f32(
                *reinterpret_cast<const uint16_t*>(p + (int64_t)g * 16 + 2 * e));
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (!(v[e] == v[e])) v[e] = -__builtin_inff();
  }
  static __device__ __forceinline__ float value(const uint32_t (&d)[4], int e) {
    if constexpr (DT == kF32) return __uint_as_float(d[e]);
    else return T16<DT == kF32 ? kBF16 : DT>::to_f32((uint16_t)(d[e >> 1] >> (16 * (e & 1))));
  }
};

constexpr float kNone = -__builtin_inff();

// 2^(j / 64)
__device__ const double kExpTable[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

// exp(x) for -40 < x <= 0, by table (P. T. P. Tang, Table-driven implementation of the
// exponential function in IEEE floating-point arithmetic, 1989): x = k ln 2 / 64 + r,
// exp(x) = 2^(k / 64) (1 + p(r)), |r| < 0.0055, p to r^5 / 120 (r^6 / 720 < 2^-54).
// Half the instructions of the library's, which has all arguments to answer for: the
// masses of 64 rows of 248320 words 29 us for 33.
__device__ __forceinline__ double exp_of(double x, const double* table) {
  const double kd0 = __builtin_fma(x, 0x1.71547652b82fep+6, 0x1.8p52);
  const int k = (int)(uint32_t)__double_as_longlong(kd0);
  const double kd = kd0 - 0x1.8p52;
  double r = __builtin_fma(kd, -0x1.62e42fefa2000p-7, x);      // ln 2 / 64 to 40 bits: exact
  r = __builtin_fma(kd, -0x1.9ef35793c7673p-47, r);
  double p = __builtin_fma(r, 1.0 / 120, 1.0 / 24);
  p = __builtin_fma(r, p, 1.0 / 6);
  p = __builtin_fma(r, p, 0.5);
  p = __builtin_fma(r * r, p, r);
  const double t = table[k & 63];
  const double y = __builtin_fma(t, p, t);
  return __longlong_as_double(__double_as_longlong(y) + ((long long)(k >> 6) << 52));
}

// Masses of a row.  w multiplies by 1 / T: within 2^-51 of the quotient, which moves a
// mass by less than its own rounding.
struct Mass {
  float m;
  double T, inv, scale;
  const double* table;                          // kExpTable, in LDS
  __device__ __forceinline__ Mass(float m_, float T_, double scale_, const double* table_)
      : m(m_), T((double)T_), inv(1.0 / (double)T_), scale(scale_), table(table_) {}
  // (l - m) / T; 0 at l = m, whatever m is
  __device__ __forceinline__ double z(float l) const {
    return l == m ? 0.0 : ((double)l - (double)m) / T;
  }
  __device__ __forceinline__ double w(float l) const {
    const double x = l == m ? 0.0 : ((double)l - (double)m) * inv;
    return x > -40.0 ? exp_of(x, table) : 0.0;  // (a NaN, inf * 0, is no mass)
  }
  // w * scale <= 2^44, rounded to an integer by adding 2^52
  __device__ __forceinline__ u64 of(double w) const {
    return (u64)__double_as_longlong(__builtin_fma(w, scale, 0x1p52)) - 0x4330000000000000ull;
  }
};

// Bin of a logit > -inf: falls with its value, by the same float steps everywhere.
__device__ __forceinline__ int bin_of(float l, float m, float per) {
  const float d = l == m ? 0.0f : (m - l) * per;
  return d < (float)(kBins - 1) ? (int)d : kBins - 1;   // (inf and NaN: the last)
}

// Larger logit, larger key (-0 as 0).
__device__ __forceinline__ uint32_t value_key(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Earlier in order, larger key.
__device__ __forceinline__ u64 order_key(float l, int i) {
  return (u64)value_key(l) << 32 | (uint32_t)~(uint32_t)i;
}
__device__ __forceinline__ float key_value(u64 k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(u64 k) { return (int)~(uint32_t)k; }

// A row's part of the workspace.
struct RowSpace {
  u64* tops;                                    // [kSampleTiles] the tiles' first words' order keys
  u64* csum;                                    // [kSampleTiles] masses of the tiles
  u64* mass;                                    // [kBins]
  u64* list;                                    // [kList] order keys
  uint32_t* count;                              // [kBins], the list's length, workgroups done
  u64* row;                                     // first word's key; the bound's bits (-inf: none)
};
__device__ __forceinline__ RowSpace row_space(void* ws, int r) {
  unsigned char* p = static_cast<unsigned char*>(ws) + (size_t)r * kSampleRowBytes;
  RowSpace s;
  s.tops = reinterpret_cast<u64*>(p);
  s.csum = s.tops + kSampleTiles;
  s.mass = s.csum + kSampleTiles;
  s.list = s.mass + kSampleBins;
  s.row = s.list + kSampleList;
  s.count = reinterpret_cast<uint32_t*>(s.row + 2);
  return s;
}

// Stores and loads at the device's coherence point, past the XCDs' own caches: what a
// workgroup reads in the launch that wrote it.
__device__ __forceinline__ void put_agent(u64* p, u64 v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 get_agent(const u64* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }

// Over the workgroup's threads, to all of them.
__device__ __forceinline__ u64 block_sum(u64 v, u64* tmp) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  v = tmp[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v += tmp[w];
  __syncthreads();
  return v;
}
// Sum over the threads before this one; total to all.
__device__ __forceinline__ u64 block_scan(u64 v, u64& total, u64* tmp) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 t = __shfl_up(s, o);
    if (lane >= o) s += t;
  }
  if (lane == 63) tmp[wave] = s;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before += tmp[w];
    total += tmp[w];
  }
  __syncthreads();
  return before + s - v;
}

// The first of chunk c's of a row's n tiles (of 2^tile granules, 64 or more: a wave's
// share at a time, whose kept mass is held apart, so that the token's is soon found).
__device__ __forceinline__ int chunk_at(int n, int c, int C) { return (int)((int64_t)n * c / C); }
template <int DT>
__device__ __forceinline__ int row_tiles(const RowView<DT>& row, int tile) {
  return (row.n + (1 << tile) - 1) >> tile;
}
// f(g) for this lane's granules of tile i
template <int DT, class F>
__device__ __forceinline__ void each_granule(const RowView<DT>& row, int tile, int i, F&& f) {
  const int g1 = min((i + 1) << tile, row.n);
  for (int g = (i << tile) + (int)(threadIdx.x & 63); g < g1; g += 64) f(g);
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max64(v, __shfl_xor(v, o));
  return v;
}

// A row's first word (order key; 0: none), and whether its list goes by the tiles' first
// words: where k of them have one.
struct Tops {
  u64 first;
  bool bound;
};
__device__ __forceinline__ Tops row_tops(const RowSet& set, const RowSpace& s, int tiles,
                                         u64* tmp) {
  u64 v = 0;
  int n = 0;
  for (int base = 0; base < tiles; base += kThreads) {
    const int i = base + (int)threadIdx.x;
    const u64 k = i < tiles ? s.tops[i] : 0;
    v = max64(v, k);
    n += __popcll(__ballot(k != 0));
  }
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) {
    tmp[threadIdx.x >> 6] = v;
    tmp[kThreads / 64 + (threadIdx.x >> 6)] = (u64)n;
  }
  __syncthreads();
  Tops t{0, false};
  n = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    t.first = max64(t.first, tmp[w]);
    n += (int)tmp[kThreads / 64 + w];
  }
  __syncthreads();
  t.bound = set.by_k && n >= set.k;
  return t;
}

// Of the upper 16 bits of value keys, the largest that k of the tiles' first words reach,
// as a logit.  One wave, PER tiles a lane (485 tiles as 8 a lane 5.4 us of step 2, as 16 7.1).
template <int PER>
__device__ __forceinline__ float bound_of(const u64* tops, int tiles, int k) {
  const int lane = threadIdx.x & 63;
  uint32_t v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    v[i] = 64 * i + lane < tiles ? (uint32_t)(tops[64 * i + lane] >> 48) : 0u;
  uint32_t bound = 0;
#pragma unroll 1
  for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
    const uint32_t x = bound | bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += __popcll(__ballot(v[i] >= x));
    if (n >= k) bound = x;
  }
  return key_value((u64)bound << 48);
}

// ---- 1: each tile's first word; the row's histogram and list are emptied -----------
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_tops_kernel(SampleArgs a, void* ws, int C) {
  const int c = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r);
  for (int i = kThreads * c + t; i < kBins; i += kThreads * C) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  if (c == 0 && t < 2) s.count[kBins + t] = 0;
  const int n = row_tiles(row, a.tile), i1 = chunk_at(n, c + 1, C);
  for (int i = chunk_at(n, c, C) + (t >> 6); i < i1; i += kThreads / 64) {
    // the largest value, then the lowest index that has it
    float top = kNone;
    int at = 0;
    each_granule(row, a.tile, i, [&](int g) {
      float v[RowView<DT>::E];
      row.load(g, v);
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        if (v[e] > top) {
          top = v[e];
          at = row.first(g) + e;
        }
      }
    });
    const u64 k = wave_max(top > kNone ? order_key(top, at) : 0);
    if ((t & 63) == 0) s.tops[i] = k;
  }
}

// ---- 2: masses ---------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_mass_kernel(SampleArgs a, void* ws, int C) {
  __shared__ u64 tmp[2 * kThreads / 64];
  __shared__ u64 hm[kBins];                     // masses, or counts
  __shared__ double table[64];
  const int c = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
  const RowSet set = row_set(a, r);
  if (set.greedy && c) return;
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r);
  const int n = row_tiles(row, a.tile), i1 = chunk_at(n, c + 1, C);
  if (t < 64) table[t] = kExpTable[t];
  const bool hist = set.by_k || set.by_p;
  if (hist)
    for (int i = t; i < kBins; i += kThreads) hm[i] = 0;
  const Tops tops = row_tops(set, s, n, tmp);   // (and the table is written)
  if (c == 0 && t < 64) {
    constexpr int PER = kSampleTiles / 64;
    const float low = !tops.bound       ? kNone
                      : n <= 32 * PER ? bound_of<PER / 2>(s.tops, n, set.k)
                                      : bound_of<PER>(s.tops, n, set.k);
    if (t == 0) {
      s.row[0] = tops.first;
      s.row[1] = __float_as_uint(low);
      if (set.greedy || !tops.first) {
        a.token[r] = tops.first ? key_index(tops.first) : -1;
        a.logprob[r] = tops.first ? 0.0f : kNone;
      }
    }
  }
  if (set.greedy || !tops.first || tops.bound) return;
  const Mass mass(key_value(tops.first), set.T, a.scale, table);
  const float per = kBinsPerNat / set.T;
  for (int i = chunk_at(n, c, C) + (t >> 6); i < i1; i += kThreads / 64) {
    u64 sum = 0;
    each_granule(row, a.tile, i, [&](int g) {
      float v[RowView<DT>::E];
      row.load(g, v);
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        if (!(v[e] > kNone)) continue;
        if (set.by_k) {
          atomicAdd(&hm[bin_of(v[e], mass.m, per)], 1ull);
          continue;
        }
        const double w = mass.w(v[e]);
        if (set.by_p) {
          const u64 W = mass.of(w);
          if (W) atomicAdd(&hm[bin_of(v[e], mass.m, per)], W);
        } else if (w >= (double)set.min_p || order_key(v[e], row.first(g) + e) == tops.first) {
          sum += mass.of(w);
        }
      }
    });
    if (!hist) {
      sum = wave_sum(sum);
      if ((t & 63) == 0) s.csum[i] = sum;
    }
  }
  if (!hist) return;
  __syncthreads();
  for (int i = t; i < kBins; i += kThreads) {
    if (!hm[i]) continue;
    if (set.by_k) atomicAdd(&s.count[i], (uint32_t)hm[i]);
    else atomicAdd(&s.mass[i], hm[i]);
  }
}

// ---- 3: the words that the cut is decided among --------------------------------------

// The words that are listed: of at least `low` (the bound); else by the cut's bin, of k
// words (the first bin up to which there are k, the last if there are fewer) or of
// p (the bin of the last word before which the mass is less than p of the whole).
struct Cut {
  int bin;                                      // -1: by low
  float low;
  u64 before, total;                            // p: mass in the bins before it, of the row
};

constexpr int kBinsPer = kBins / kThreads;      // a thread's bins
__device__ __forceinline__ Cut find_cut(const RowSet& set, const RowSpace& s, float low, u64* tmp,
                                        Cut* out) {
  if (low > kNone) return Cut{-1, low, 0, 0};
  u64 v[kBinsPer], sum = 0, all;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    const int bin = (int)threadIdx.x * kBinsPer + i;
    v[i] = set.by_k ? s.count[bin] : s.mass[bin];
    sum += v[i];
  }
  u64 b = block_scan(sum, all, tmp);            // words, or mass, before the bins
  const u64 k = (u64)set.k < all ? (u64)set.k : all;
  const double goal = (double)set.p * (double)all;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    const int bin = (int)threadIdx.x * kBinsPer + i;
    // p: the first bin that reaches the goal (later ones start beyond it)
    if (set.by_k ? b < k && b + v[i] >= k : (double)b < goal && (double)(b + v[i]) >= goal)
      *out = Cut{bin, 0.0f, b, all};
    b += v[i];
  }
  __syncthreads();
  return *out;
}

// Chunk c's words onto the list (whose length counts on past kList), and for p the mass
// of its tiles before the cut.  SKIP: a tile whose first word lies behind the cut, which has
// nothing to list or add, is not read (64 rows of 248320 words 19.2 for 19.6 us; with few
// rows the look at that word is one more step of the chain, 0.5 us).
template <int DT, bool SKIP>
__device__ __forceinline__ void list_words(const SampleArgs& a, const RowView<DT>& row,
                                           const RowSet& set, const RowSpace& s, const Cut& cut,
                                           const Mass& mass, u64 first, int c, int C) {
  const float per = kBinsPerNat / set.T;
  const int t = threadIdx.x, tiles = row_tiles(row, a.tile), i1 = chunk_at(tiles, c + 1, C);
  for (int i = chunk_at(tiles, c, C) + (t >> 6); i < i1; i += kThreads / 64) {
    if constexpr (SKIP) {
      const u64 top = s.tops[i];
      if (!top || (cut.bin < 0 ? key_value(top) < cut.low
                               : bin_of(key_value(top), mass.m, per) > cut.bin)) {
        if (!set.by_k && (t & 63) == 0) put_agent(&s.csum[i], (u64)0);
        continue;
      }
    }
    u64 sum = 0;
    each_granule(row, a.tile, i, [&](int g) {
      float v[RowView<DT>::E];
      row.load(g, v);
      uint32_t mine = 0;                        // its words that are listed
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        bool listed = v[e] >= cut.low;
        if (cut.bin >= 0) {
          const int b = bin_of(v[e], mass.m, per);
          listed = v[e] > kNone && (b == cut.bin || (set.by_k && b < cut.bin));
          if (!set.by_k && b < cut.bin) {
            const double w = mass.w(v[e]);
            if (w >= (double)set.min_p || order_key(v[e], row.first(g) + e) == first)
              sum += mass.of(w);
          }
        }
        mine |= (uint32_t)listed << e;
      }
      // the wave's places on the list by one atomic, whose answer takes a microsecond
      if (!__ballot(mine != 0)) return;
      uint32_t n = 0, before[RowView<DT>::E];
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        const u64 b = __ballot(mine >> e & 1);
        before[e] = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32),
                                                  __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
        n += __popcll(b);
      }
      uint32_t at = 0;
      if ((t & 63) == (int)__builtin_ctzll(__ballot(true))) at = atomicAdd(&s.count[kBins], n);
      at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e)
        if ((mine >> e & 1) && at + before[e] < kList)
          put_agent(&s.list[at + before[e]], order_key(v[e], row.first(g) + e));
    });
    if (!set.by_k) {
      sum = wave_sum(sum);
      if ((t & 63) == 0) put_agent(&s.csum[i], sum);
    }
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_list_kernel(SampleArgs a, void* ws, int C) {
  __shared__ u64 tmp[2 * kThreads / 64];
  __shared__ double table[64];
  __shared__ Cut shared_cut;
  const int r = blockIdx.y, t = threadIdx.x;
  const RowSet set = row_set(a, r);
  if (set.greedy || !(set.by_k || set.by_p)) return;
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r);
  const u64 first = s.row[0];
  const float low = __uint_as_float((uint32_t)s.row[1]);
  if (!first) return;
  if (t < 64) table[t] = kExpTable[t];
  const Mass mass(key_value(first), set.T, a.scale, table);
  const Cut cut = find_cut(set, s, low, tmp, &shared_cut);
  __syncthreads();                              // the table is written
  list_words<DT, true>(a, row, set, s, cut, mass, first, blockIdx.x, C);
}

// ---- 4: the token ------------------------------------------------------------------

// u of the kept mass, as a place in it.
__device__ __forceinline__ u64 place(float u, u64 S) {
  const double x = (double)u * (double)S;
  if (!(x > 0.0)) return 0;
  const u64 t = x < 0x1p63 ? (u64)x : S;
  return t < S ? t : S - 1;
}

struct Pick {
  int token;
  float logit;
};

// Which words are kept: the first, and those of at least min_p that do not come after
// `end` (an order key).
struct Kept {
  u64 first, end;
  double min_p;
  __device__ __forceinline__ bool operator()(u64 key, double w) const {
    return key == first || (w >= min_p && key >= end);
  }
};

// The kept mass of this thread's granules among [g0, g1).
template <int DT>
__device__ __forceinline__ u64 kept_mass(const RowView<DT>& row, const Mass& mass, int g,
                                         const Kept& kept, float (&v)[RowView<DT>::E],
                                         u64 (&W)[RowView<DT>::E]) {
  u64 sum = 0;
  row.load(g, v);
#pragma unroll
  for (int e = 0; e < RowView<DT>::E; ++e) {
    const double w = mass.w(v[e]);
    W[e] = v[e] > kNone && kept(order_key(v[e], row.first(g) + e), w) ? mass.of(w) : 0;
    sum += W[e];
  }
  return sum;
}

// The kept word of granules [g0, g1) that place t (of their kept mass) falls on.
template <int DT>
__device__ __forceinline__ void pick_in(const RowView<DT>& row, const Mass& mass, int g0, int g1,
                                        u64 t, const Kept& kept, u64* tmp, Pick* out) {
  u64 run = 0;
  for (int base = g0; base < g1; base += kThreads) {
    const int g = base + (int)threadIdx.x;
    float v[RowView<DT>::E];
    u64 W[RowView<DT>::E], sum = 0, all;
    if (g < g1) sum = kept_mass<DT>(row, mass, g, kept, v, W);
    const u64 before = run + block_scan(sum, all, tmp);
    if (g < g1 && before <= t && t < before + sum) {
      u64 b = before;
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        if (b <= t && t < b + W[e]) *out = Pick{row.first(g) + e, v[e]};
        b += W[e];
      }
    }
    run += all;
    if (t < run) break;                         // uniform
  }
  __syncthreads();
}

// The order key of the last word kept by k words (by_mass false) or by mass goal, and
// the mass up to it, by radix over value keys and then indexes: the words whose key's
// top bits equal the prefix are counted by their next 8 bits.
template <int DT>
__device__ __noinline__ u64 select_key(const RowView<DT>& row, const Mass& mass, bool by_mass,
                                       u64 k, double goal, u64& upto, u64* hm, uint32_t* hc,
                                       u64* tmp, u64* res) {
  u64 prefix = 0, cb = 0, mb = 0;               // counts and mass before the prefix's words
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      hm[i] = 0;
      hc[i] = 0;
    }
    __syncthreads();
    for (int g = threadIdx.x; g < row.n; g += kThreads) {
      float v[RowView<DT>::E];
      row.load(g, v);
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        if (!(v[e] > kNone)) continue;
        const u64 key = order_key(v[e], row.first(g) + e);
        if (shift < 56 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        const int b = 255 - (int)(key >> shift & 255);
        atomicAdd(&hc[b], 1u);
        const u64 W = mass.of(mass.w(v[e]));
        if (W) atomicAdd(&hm[b], W);
      }
    }
    __syncthreads();
    const int t = threadIdx.x;
    const u64 m = t < 256 ? hm[t] : 0, n = t < 256 ? hc[t] : 0;
    u64 all;
    const u64 m0 = mb + block_scan(m, all, tmp);
    const u64 c0 = cb + block_scan(n, all, tmp);
    const bool here = n && (by_mass ? (double)m0 < goal && (double)(m0 + m) >= goal
                                    : c0 < k && c0 + n >= k);
    if (here) {
      res[0] = prefix | (u64)(255 - t) << shift;
      res[1] = c0;
      res[2] = m0;
      res[3] = m0 + m;
    }
    __syncthreads();
    prefix = res[0];
    cb = res[1];
    mb = res[2];
    upto = res[3];
    __syncthreads();
  }
  return prefix;
}

// keys[0 .. n - 1] into falling order; tmp: n places, and n counts.
//  * Up to 256 keys: a key's place is the number of larger ones, counted by all pairs,
//    those of a key by 512 / P threads (P: n raised to a power of two, 64 at least).
//  * More: a bitonic network over P (places past n are 0).  Pairs of places up to 64
//    apart are a wave's own, 128 places of it, and its LDS instructions run in order: no
//    barrier.  (A step takes 0.2 us; of 64 keys 4.2 us in its 21 steps, 0.9 by pairs.)
__device__ __forceinline__ void sort_falling(u64* keys, int n, u64* tmp, uint32_t* places) {
  int P = 64;
  while (P < n) P <<= 1;
  if (P <= 256) {
    const int t = threadIdx.x, i = t & (P - 1), parts = kThreads / P;
    if (t < P) places[t] = 0;
    __syncthreads();
    if (i < n) {
      const u64 key = keys[i];
      uint32_t larger = 0;
#pragma unroll 4
      for (int j = t / P; j < n; j += parts) larger += keys[j] > key;
      atomicAdd(&places[i], larger);
    }
    __syncthreads();
    if (t < n) tmp[places[t]] = keys[t];
    __syncthreads();
    if (t < n) keys[t] = tmp[t];
    __syncthreads();
    return;
  }
  for (int i = n + (int)threadIdx.x; i < P; i += kThreads) keys[i] = 0;
  __syncthreads();
  for (int k = 2; k <= P; k <<= 1) {
    for (int j = k >> 1; j; j >>= 1) {
      // thread t takes pair (i, i | j): bit j of i is left out of t
      for (int t = (int)threadIdx.x; t < P / 2; t += kThreads) {
        const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1));
        const u64 x = keys[i], y = keys[i | j];
        if ((x < y) == ((i & k) == 0)) {
          keys[i] = y;
          keys[i | j] = x;
        }
      }
      const int next = j > 1 ? j >> 1 : k;
      if (j > 64 || next > 64) {
        __syncthreads();
      } else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
    }
  }
  __syncthreads();
}

// Of n keys, the last in falling order before which the mass (from `before` on) is less
// than goal, up to which it is not: by the 11 highest bits in which those still asked
// about differ (bins: 2048 masses), until one is left.  Keys of a bin of a p row have
// few values, and differ in the index's 18 bits: three rounds of 1.5 us, where sorting
// 2048 took 16.
__device__ __forceinline__ u64 cut_of_list(const u64* keys, int n, u64* bins, const Mass& mass,
                                           u64 before, double goal, u64* tmp, u64* res) {
  const int t = threadIdx.x;
  u64 prefix = 0;
  int top = 64;                                 // asked about: keys with prefix's bits from top on
  auto asked = [&](u64 key) { return top == 64 || key >> top == prefix >> top; };
#pragma unroll 1
  for (;;) {
    u64 ones = 0, zeros = 0;                    // bits that are one, or zero, in any
#pragma unroll 1
    for (int i = t; i < n; i += kThreads) {
      const u64 key = keys[i];
      if (asked(key)) {
        ones |= key;
        zeros |= ~key;
      }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      ones |= __shfl_xor(ones, o);
      zeros |= __shfl_xor(zeros, o);
    }
    if ((t & 63) == 0) {
      tmp[t >> 6] = ones;
      tmp[kThreads / 64 + (t >> 6)] = zeros;
    }
    for (int i = t; i < kBins; i += kThreads) bins[i] = 0;
    if (t == 0) res[0] = res[1] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      ones |= tmp[w];
      zeros |= tmp[kThreads / 64 + w];
    }
    const u64 differ = ones & zeros;
    if (!differ) return ones;                   // one key
    const int high = 63 - __builtin_clzll(differ), shift = high > 10 ? high - 10 : 0;
#pragma unroll 1
    for (int i = t; i < n; i += kThreads) {
      const u64 key = keys[i];
      if (asked(key)) atomicAdd(&bins[kBins - 1 - (key >> shift & (kBins - 1))],
                                mass.of(mass.w(key_value(key))));
    }
    __syncthreads();
    u64 v[kBinsPer], sum = 0, all;
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) sum += v[i] = bins[t * kBinsPer + i];
    u64 b = before + block_scan(sum, all, tmp);
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) {
      if ((double)b < goal && (double)(b + v[i]) >= goal) {
        res[0] = (u64)(kBins - 1 - (t * kBinsPer + i));
        res[1] = b;
      }
      b += v[i];
    }
    __syncthreads();
    // the bits above the 11 are those of all that were asked about
    prefix = ((ones >> shift & ~(u64)(kBins - 1)) | res[0]) << shift;
    before = res[1];
    top = shift;
    __syncthreads();
  }
}

// LIST: step 3 as well, by C workgroups per row; else one per row.
template <int DT, bool LIST>
__global__ __launch_bounds__(kThreads, 4) void sample_pick_kernel(SampleArgs a, void* ws, int C) {
  __shared__ u64 tmp[2 * kThreads / 64];
  __shared__ u64 keys[kList];
  __shared__ u64 masses[kList];
  __shared__ u64 part[kSampleTiles];            // the tiles' kept masses
  __shared__ double table[64];
  __shared__ Cut shared_cut;
  __shared__ Pick pick;
  __shared__ u64 res[4], left;
  __shared__ int at, last_done;
  __shared__ u64 hm[256];
  __shared__ uint32_t hc[256];
  const int c = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
  const RowSet set = row_set(a, r);
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r);
  const int tiles = row_tiles(row, a.tile);
  const bool list = set.by_k || set.by_p;
  const u64 first = s.row[0];
  const float low = __uint_as_float((uint32_t)s.row[1]);
  if (set.greedy || !first || (!list && c)) return;       // (step 2 wrote those)
  if (t < 64) table[t] = kExpTable[t];
  __syncthreads();
  const Mass mass(key_value(first), set.T, a.scale, table);
  const double min_p = (double)set.min_p;
  Cut cut{-1, 0.0f, 0, 0};
  int n = 0;
  if (list) {
    if (LIST || !set.by_k) cut = find_cut(set, s, low, tmp, &shared_cut);
    if constexpr (LIST) {
      list_words<DT, false>(a, row, set, s, cut, mass, first, c, C);
      // the last of the row's workgroups goes on, with what the others wrote: each
      // wave's stores are made before its workgroup counts itself
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (t == 0) last_done = atomicAdd(&s.count[kBins + 1], 1u) == (uint32_t)(C - 1);
      __syncthreads();
      if (!last_done) return;
    }
    n = (int)__hip_atomic_load(&s.count[kBins], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const bool whole = n <= kList;                // the list is
  if (t == 0) pick = Pick{key_index(first), mass.m};
  u64 S = 0, place_at;
  Kept kept{first, 0, min_p};
  if (list && whole) {
    for (int i = t; i < n; i += kThreads) keys[i] = get_agent(&s.list[i]);
    __syncthreads();
  }
  if (list && whole && !set.by_k) {
    // the bins before the cut's are in the tiles' sums; its kept words join theirs (words
    // of the bins before it precede the last word that p keeps)
    kept.end = cut_of_list(keys, n, masses, mass, cut.before, (double)set.p * (double)cut.total,
                           tmp, res);
    for (int i = t; i < tiles; i += kThreads) part[i] = get_agent(&s.csum[i]);
    __syncthreads();
#pragma unroll 1
    for (int i = t; i < n; i += kThreads) {
      const double w = mass.w(key_value(keys[i]));
      if (kept(keys[i], w))
        atomicAdd(&part[(key_index(keys[i]) + row.off) / RowView<DT>::E >> a.tile], mass.of(w));
    }
    __syncthreads();
  } else if (list && whole) {
    sort_falling(keys, n, masses, hc);
    // the kept words are a prefix: of k, of those before which p's mass is not reached,
    // and of those of min_p
    const int nk = set.k < n ? set.k : n;
    uint32_t of_p = 0, of_min = 0;
#pragma unroll 1
    for (int i = t; i < nk; i += kThreads) {
      const double w = mass.w(key_value(keys[i]));
      masses[i] = mass.of(w);
      of_min += w >= min_p || keys[i] == first;
    }
    __syncthreads();
    // thread t has the `per` places from t per
    auto scan = [&](int m, int per, u64& total) {
      u64 sum = 0;
#pragma unroll 1
      for (int i = t * per; i < (t + 1) * per && i < m; ++i) sum += masses[i];
      return block_scan(sum, total, tmp);
    };
    int per = (nk + kThreads - 1) / kThreads;
    u64 total;
    u64 b = scan(nk, per, total);
    const double goal = (double)set.p * (double)total;
#pragma unroll 1
    for (int i = t * per; i < (t + 1) * per && i < nk; ++i) {
      of_p += !set.by_p || (double)b < goal || keys[i] == first;
      b += masses[i];
    }
    const u64 both = block_sum((u64)of_p << 32 | of_min, tmp);
    const int kept_p = (int)(both >> 32);
    const int m = min(kept_p, (int)(uint32_t)both);
    // the kept words in index order (the index, complemented in the key already, above
    // the value), and the one whose share holds the place
#pragma unroll 1
    for (int i = t; i < m; i += kThreads) keys[i] = keys[i] << 32 | keys[i] >> 32;
    sort_falling(keys, m, masses, hc);
#pragma unroll 1
    for (int i = t; i < m; i += kThreads)
      masses[i] = mass.of(mass.w(key_value(keys[i] << 32)));
    __syncthreads();
    per = (m + kThreads - 1) / kThreads;
    b = scan(m, per, S);
    place_at = place(set.u, S);
#pragma unroll 1
    for (int i = t * per; i < (t + 1) * per && i < m; ++i) {
      if (b <= place_at && place_at < b + masses[i])
        pick = Pick{key_index(keys[i] >> 32), key_value(keys[i] << 32)};
      b += masses[i];
    }
  } else if (list) {
    // too many to list: the cut by radix over the row
    u64 upto = 0;
    double total = (double)cut.total;
    if (set.by_k) {
      // (the words of a bound's row are more than k)
      u64 k = set.k, all = 0;
      if (!(low > kNone)) {
        for (int b = t; b < kBins; b += kThreads) all += s.count[b];
        all = block_sum(all, tmp);
        k = k < all ? k : all;
      }
      kept.end = select_key<DT>(row, mass, false, k, 0.0, upto, hm, hc, tmp, res);
      total = (double)upto;
    }
    if (set.by_p)
      kept.end = select_key<DT>(row, mass, true, 0, (double)set.p * total, upto, hm, hc, tmp, res);
#pragma unroll 1
    for (int i = t >> 6; i < tiles; i += kThreads / 64) {
      u64 sum = 0;
      each_granule(row, a.tile, i, [&](int g) {
        float v[RowView<DT>::E];
        u64 W[RowView<DT>::E];
        sum += kept_mass<DT>(row, mass, g, kept, v, W);
      });
      sum = wave_sum(sum);
      if ((t & 63) == 0) part[i] = sum;
    }
    __syncthreads();
  } else {
    for (int i = t; i < tiles; i += kThreads) part[i] = s.csum[i];
    __syncthreads();
  }
  if (!set.by_k || !whole) {
    // the tile that holds the place, then the word in it
    const int per = (tiles + kThreads - 1) / kThreads;
    u64 sum = 0;
    for (int i = t * per; i < (t + 1) * per && i < tiles; ++i) sum += part[i];
    u64 b = block_scan(sum, S, tmp);
    place_at = place(set.u, S);
    for (int i = t * per; i < (t + 1) * per && i < tiles; ++i) {
      if (b <= place_at && place_at < b + part[i]) {
        at = i;
        left = place_at - b;
      }
      b += part[i];
    }
    __syncthreads();
    pick_in<DT>(row, mass, at << a.tile, min((at + 1) << a.tile, row.n), left, kept, tmp, &pick);
  }
  __syncthreads();
  if (t == 0) {
    a.token[r] = pick.token;
    a.logprob[r] = (float)(mass.z(pick.logit) - log((double)S / a.scale));
  }
}

}  // namespace

int launch_sample(const SampleArgs& a0, int dtype, void* ws, hipStream_t st, int* nlaunch) {
  const int size = dtype == kF32 ? 4 : 2;
  for (int64_t r0 = 0; r0 < a0.R; r0 += kSampleRows) {
    SampleArgs a = a0;
    a.R = a0.R - r0 < kSampleRows ? a0.R - r0 : kSampleRows;
    a.logits = static_cast<const unsigned char*>(a0.logits) + r0 * a0.row_stride * size;
    a.u += r0;
    if (a.temperature) a.temperature += r0;
    if (a.top_k) a.top_k += r0;
    if (a.top_p) a.top_p += r0;
    if (a.min_p) a.min_p += r0;
    a.token += r0;
    a.logprob += r0;
    const int C = sample_chunks(a0.R, a.V);
    // steps 3 and 4 in one where all workgroups of step 4's size run at once
    const bool one = C * a.R <= 2 * device_cu_count();
    a.tile = sample_tile(a.V, dtype);
    const dim3 grid((unsigned)C, (unsigned)a.R);
    auto go = [&](auto dtc) {
      constexpr int DT = decltype(dtc)::value;
      hipLaunchKernelGGL(sample_tops_kernel<DT>, grid, dim3(kThreads), 0, st, a, ws, C);
      hipLaunchKernelGGL(sample_mass_kernel<DT>, grid, dim3(kThreads), 0, st, a, ws, C);
      if (one) {
        hipLaunchKernelGGL((sample_pick_kernel<DT, true>), grid, dim3(kThreads), 0, st, a, ws, C);
      } else {
        hipLaunchKernelGGL(sample_list_kernel<DT>, grid, dim3(kThreads), 0, st, a, ws, C);
        hipLaunchKernelGGL((sample_pick_kernel<DT, false>), dim3(1, (unsigned)a.R),
                           dim3(kThreads), 0, st, a, ws, 1);
      }
    };
    if (dtype == kBF16) go(std::integral_constant<int, kBF16>{});
    else if (dtype == kF16) go(std::integral_constant<int, kF16>{});
    else go(std::integral_constant<int, kF32>{});
    *nlaunch += one ? 3 : 4;
  }
  return 0;
}

}  // namespace mq
