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
// row is spread over workgroups (chunks), and the passes are launches of one
// sequence, for all rows whatever their settings:
//   1 each chunk's largest logit (and its index);
//   2 masses: rows without k and p, each chunk's kept mass; the others, a histogram of
//     counts (and without k, masses) over 2048 bins of (m - l) / T, 1/64 wide;
//   3 rows with k or p: the bin in which the cut falls, from the histogram (k: the whole
//     list of words up to that bin, a few hundred; p: that bin's words), and for p
//     each chunk's mass in the bins before it;
//   4 one workgroup per row: the cut among the listed words, by comparing all pairs (no
//     sort: a word's rank and the mass before it are sums over the words that precede
//     it), the chunk and the word that u points at.
// A list of more than 4096 words (many equal logits, k in the thousands) is not made:
// step 4 then selects by radix over the row.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mq_common.h"
#include "sample_launch.h"

namespace mq {

namespace {

constexpr int kBins = 2048;
constexpr float kBinsPerNat = 64.0f;            // bins cover 32 nats, past which masses are 0
constexpr int kList = 4096;                     // listed words of a row
constexpr int kPassThreads = 256, kPickThreads = 1024;

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

// The row's largest logit, inverse temperature's place and mass scale.
struct Mass {
  float m;
  double T, scale;
  // (l - m) / T; 0 at l = m, whatever m is
  __device__ __forceinline__ double z(float l) const {
    return l == m ? 0.0 : ((double)l - (double)m) / T;
  }
  __device__ __forceinline__ double w(float l) const {
    const double x = z(l);
    return x > -40.0 ? exp(x) : 0.0;            // (a NaN, inf / inf, is no mass)
  }
  __device__ __forceinline__ u64 of(double w) const { return (u64)(w * scale + 0.5); }
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
  u64* cmax;                                    // [C] order keys
  u64* csum;                                    // [C]
  u64* mass;                                    // [kBins]
  u64* list;                                    // [kList] order keys
  uint32_t* count;                              // [kBins], then the list's length
};
__device__ __forceinline__ RowSpace row_space(void* ws, int r, int C) {
  unsigned char* p = static_cast<unsigned char*>(ws) + (size_t)r * sample_row_bytes(C);
  RowSpace s;
  s.cmax = reinterpret_cast<u64*>(p);
  s.csum = s.cmax + C;
  s.mass = s.csum + C;
  s.list = s.mass + kBins;
  s.count = reinterpret_cast<uint32_t*>(s.list + kList);
  return s;
}

__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }

// Over the workgroup's NT threads, to all of them.
template <int NT>
__device__ __forceinline__ u64 block_max(u64 v, u64* tmp) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max64(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  v = tmp[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = max64(v, tmp[w]);
  __syncthreads();
  return v;
}
template <int NT>
__device__ __forceinline__ u64 block_sum(u64 v, u64* tmp) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  v = tmp[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v += tmp[w];
  __syncthreads();
  return v;
}
// Sum over the threads before this one; total to all.
template <int NT>
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
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) before += tmp[w];
    total += tmp[w];
  }
  __syncthreads();
  return before + s - v;
}

// Chunk c of a row's n granules.
__device__ __forceinline__ int chunk_at(int n, int c, int C) { return (int)((int64_t)n * c / C); }

// The first word of the row (order key), from the chunks'; 0: none.
template <int NT>
__device__ __forceinline__ u64 row_first(const RowSpace& s, int C, u64* tmp) {
  u64 v = 0;
  for (int c = threadIdx.x; c < C; c += NT) v = max64(v, s.cmax[c]);
  return block_max<NT>(v, tmp);
}

// ---- 1: each chunk's first word; the row's histogram and list are emptied ----------
template <int DT>
__global__ __launch_bounds__(kPassThreads) void sample_max_kernel(SampleArgs a, void* ws, int C) {
  __shared__ u64 tmp[kPassThreads / 64];
  const int c = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r, C);
  for (int i = kPassThreads * c + t; i < kBins; i += kPassThreads * C) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  if (c == 0 && t == 0) s.count[kBins] = 0;
  const int g1 = chunk_at(row.n, c + 1, C);
  u64 best = 0;
  for (int g = chunk_at(row.n, c, C) + t; g < g1; g += kPassThreads) {
    float v[RowView<DT>::E];
    row.load(g, v);
#pragma unroll
    for (int e = 0; e < RowView<DT>::E; ++e)
      if (v[e] > kNone) best = max64(best, order_key(v[e], row.first(g) + e));
  }
  best = block_max<kPassThreads>(best, tmp);
  if (t == 0) s.cmax[c] = best;
}

// ---- 2: masses ---------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(kPassThreads) void sample_mass_kernel(SampleArgs a, void* ws, int C) {
  __shared__ u64 tmp[kPassThreads / 64];
  __shared__ u64 hm[kBins];
  __shared__ uint32_t hc[kBins];
  const int c = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
  const RowSet set = row_set(a, r);
  if (set.greedy) return;
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r, C);
  const u64 first = row_first<kPassThreads>(s, C, tmp);
  if (!first) return;
  const Mass mass{key_value(first), (double)set.T, a.scale};
  const bool hist = set.by_k || set.by_p;
  if (hist) {
    for (int i = t; i < kBins; i += kPassThreads) {
      hm[i] = 0;
      hc[i] = 0;
    }
    __syncthreads();
  }
  const float per = kBinsPerNat / set.T;
  const int g1 = chunk_at(row.n, c + 1, C);
  u64 sum = 0;
  for (int g = chunk_at(row.n, c, C) + t; g < g1; g += kPassThreads) {
    float v[RowView<DT>::E];
    row.load(g, v);
#pragma unroll
    for (int e = 0; e < RowView<DT>::E; ++e) {
      if (!(v[e] > kNone)) continue;
      if (hist) {
        const int b = bin_of(v[e], mass.m, per);
        atomicAdd(&hc[b], 1u);
        if (!set.by_k) atomicAdd(&hm[b], mass.of(mass.w(v[e])));   // (k: of the listed words alone)
        continue;
      }
      const double w = mass.w(v[e]);
      if (w >= (double)set.min_p || order_key(v[e], row.first(g) + e) == first) sum += mass.of(w);
    }
  }
  if (!hist) {
    sum = block_sum<kPassThreads>(sum, tmp);
    if (t == 0) s.csum[c] = sum;
    return;
  }
  __syncthreads();
  for (int i = t; i < kBins; i += kPassThreads) {
    if (hc[i]) {
      atomicAdd(&s.count[i], hc[i]);
      if (hm[i]) atomicAdd(&s.mass[i], hm[i]);
    }
  }
}

// The bin of the cut.  by_k: the first bin up to which there are k words, the last
// bin if there are fewer; else the bin of the last word before which the mass is less
// than p of the whole.
struct Cut {
  int bin;
  u64 before;                                   // mass in the bins before it
  u64 total;                                    // of the row
  uint32_t words;                               // by_k: up to the bin; else in it
};
template <int NT>
__device__ __forceinline__ Cut find_cut(const RowSet& set, const RowSpace& s, u64* tmp, Cut* out) {
  constexpr int PER = kBins / NT;
  const int b0 = threadIdx.x * PER;
  u64 m[PER], ms = 0, cs = 0, all, words;
  uint32_t n[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    m[i] = s.mass[b0 + i];
    n[i] = s.count[b0 + i];
    ms += m[i];
    cs += n[i];
  }
  u64 mb = block_scan<NT>(ms, all, tmp);
  u64 cb = block_scan<NT>(cs, words, tmp);
  const double goal = (double)set.p * (double)all;
  if (threadIdx.x == 0) *out = Cut{-1, 0, all, 0};
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (n[i]) {
      if (set.by_k) {
        const u64 k = (u64)set.k < words ? (u64)set.k : words;
        if (cb < k && cb + n[i] >= k) *out = Cut{b0 + i, mb, all, (uint32_t)(cb + n[i])};
      } else if ((double)mb < goal && (double)(mb + m[i]) >= goal) {
        // the first bin that reaches the goal (later ones start beyond it)
        *out = Cut{b0 + i, mb, all, n[i]};
      }
    }
    mb += m[i];
    cb += n[i];
  }
  __syncthreads();
  const Cut cut = *out;
  __syncthreads();
  return cut;
}

// ---- 3: the words that the cut is decided among ------------------------------------
template <int DT>
__global__ __launch_bounds__(kPassThreads) void sample_list_kernel(SampleArgs a, void* ws, int C) {
  __shared__ u64 tmp[kPassThreads / 64];
  __shared__ Cut shared_cut;
  const int c = blockIdx.x, r = blockIdx.y, t = threadIdx.x;
  const RowSet set = row_set(a, r);
  if (set.greedy || !(set.by_k || set.by_p)) return;
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r, C);
  const u64 first = row_first<kPassThreads>(s, C, tmp);
  if (!first) return;
  const Mass mass{key_value(first), (double)set.T, a.scale};
  const Cut cut = find_cut<kPassThreads>(set, s, tmp, &shared_cut);
  if (cut.words > kList) return;
  const float per = kBinsPerNat / set.T;
  const int g1 = chunk_at(row.n, c + 1, C);
  u64 sum = 0;
  for (int g = chunk_at(row.n, c, C) + t; g < g1; g += kPassThreads) {
    float v[RowView<DT>::E];
    row.load(g, v);
#pragma unroll
    for (int e = 0; e < RowView<DT>::E; ++e) {
      if (!(v[e] > kNone)) continue;
      const int b = bin_of(v[e], mass.m, per);
      if (b == cut.bin || (set.by_k && b < cut.bin)) {
        const uint32_t at = atomicAdd(&s.count[kBins], 1u);
        if (at < kList) s.list[at] = order_key(v[e], row.first(g) + e);
      } else if (b < cut.bin) {
        const double w = mass.w(v[e]);
        if (w >= (double)set.min_p || order_key(v[e], row.first(g) + e) == first)
          sum += mass.of(w);
      }
    }
  }
  if (set.by_k) return;
  sum = block_sum<kPassThreads>(sum, tmp);
  if (t == 0) s.csum[c] = sum;
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

// The kept word of granules [g0, g1) that place t (of their kept mass) falls on;
// kept(key, w): whether a word is kept.
template <int DT, class Kept>
__device__ __forceinline__ void pick_in(const RowView<DT>& row, const Mass& mass, int g0, int g1,
                                        u64 t, Kept kept, u64* tmp, Pick* out) {
  u64 run = 0;
  for (int base = g0; base < g1; base += kPickThreads) {
    const int g = base + (int)threadIdx.x;
    float v[RowView<DT>::E];
    u64 W[RowView<DT>::E], sum = 0, all;
    if (g < g1) {
      row.load(g, v);
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        W[e] = 0;
        if (v[e] > kNone) {
          const double w = mass.w(v[e]);
          if (kept(order_key(v[e], row.first(g) + e), w)) W[e] = mass.of(w);
        }
        sum += W[e];
      }
    }
    const u64 before = run + block_scan<kPickThreads>(sum, all, tmp);
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

// The chunk (of at most kPickThreads) whose kept mass holds t; t becomes the place in it.
__device__ __forceinline__ int pick_chunk(const u64* csum, int C, u64& t, u64* tmp, int* at,
                                          u64* left) {
  if (threadIdx.x == 0) *at = -1;
  __syncthreads();
  const int c0 = (int)threadIdx.x;
  const u64 v = c0 < C ? csum[c0] : 0;
  u64 all;
  const u64 before = block_scan<kPickThreads>(v, all, tmp);
  if (before <= t && t < before + v) {
    *at = c0;
    *left = t - before;
  }
  __syncthreads();
  const int c = *at;
  t = *left;
  __syncthreads();
  return c;
}

// The order key of the last word kept by k words (by_mass false) or by mass goal, and
// the mass up to it, by radix over value keys and then indexes: the words whose key's
// top bits equal the prefix are counted by their next 8 bits.
template <int DT>
__device__ u64 select_key(const RowView<DT>& row, const Mass& mass, bool by_mass, u64 k,
                          double goal, u64& upto, u64* hm, uint32_t* hc, u64* tmp, u64* res) {
  u64 prefix = 0, cb = 0, mb = 0;               // counts and mass before the prefix's words
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kPickThreads) {
      hm[i] = 0;
      hc[i] = 0;
    }
    __syncthreads();
    for (int g = threadIdx.x; g < row.n; g += kPickThreads) {
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
    const u64 m0 = mb + block_scan<kPickThreads>(m, all, tmp);
    const u64 c0 = cb + block_scan<kPickThreads>(n, all, tmp);
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

template <int DT>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a, void* ws, int C) {
  __shared__ u64 tmp[kPickThreads / 64];
  __shared__ u64 keys[kList];
  __shared__ u64 masses[kList];
  __shared__ u64 chunks[kPickThreads];
  __shared__ Cut shared_cut;
  __shared__ Pick pick;
  __shared__ u64 res[4], left, cutkey;
  __shared__ int at;
  __shared__ u64 hm[256];
  __shared__ uint32_t hc[256];
  const int r = blockIdx.x, t = threadIdx.x;
  const RowSet set = row_set(a, r);
  const RowView<DT> row(a, r);
  const RowSpace s = row_space(ws, r, C);
  const u64 first = row_first<kPickThreads>(s, C, tmp);
  if (set.greedy || !first) {
    if (t == 0) {
      a.token[r] = first ? key_index(first) : -1;
      a.logprob[r] = first ? 0.0f : kNone;
    }
    return;
  }
  const Mass mass{key_value(first), (double)set.T, a.scale};
  if (t == 0) pick = Pick{key_index(first), mass.m};
  const double min_p = (double)set.min_p;
  u64 S = 0, place_at;
  const bool hist = set.by_k || set.by_p;
  Cut cut{-1, 0, 0, 0};
  if (hist) cut = find_cut<kPickThreads>(set, s, tmp, &shared_cut);
  if (hist && cut.words <= kList) {
    const int n = (int)cut.words;
    for (int i = t; i < n; i += kPickThreads) {
      keys[i] = s.list[i];
      masses[i] = mass.of(mass.w(key_value(keys[i])));
    }
    __syncthreads();
    // rank of each listed word and the mass before it; for k, only the first k count
    constexpr int PER = kList / kPickThreads;
    u64 before[PER], kmass = 0;
    bool in[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int i = q * kPickThreads + t;
      before[q] = set.by_k ? 0 : cut.before;
      in[q] = i < n;
      if (!in[q]) continue;
      const u64 key = keys[i];
      int rank = 0;
      u64 m = 0;
      for (int j = 0; j < n; ++j) {
        const bool lead = keys[j] > key;
        rank += lead;
        m += lead ? masses[j] : 0;
      }
      before[q] += m;
      if (set.by_k) {
        in[q] = rank < set.k;
        if (in[q]) kmass += masses[i];
      }
    }
    const u64 total = set.by_k ? block_sum<kPickThreads>(kmass, tmp) : cut.total;
    const double goal = (double)set.p * (double)total;
    u64 sum = 0, last = ~0ull;                  // the last word kept by k and p has the smallest key
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int i = q * kPickThreads + t;
      if (!in[q]) continue;
      const bool lead = keys[i] == first;
      if (set.by_p) in[q] = lead || (double)before[q] < goal;
      if (in[q]) last = last < keys[i] ? last : keys[i];
      if (in[q]) in[q] = lead || mass.w(key_value(keys[i])) >= min_p;
      if (in[q]) sum += masses[i];
    }
    __syncthreads();
    if (set.by_k) {
      // all kept words are listed: the one whose share in index order holds the place
      S = block_sum<kPickThreads>(sum, tmp);
      place_at = place(set.u, S);
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int i = q * kPickThreads + t;
        if (i < n && !in[q]) masses[i] = 0;
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int i = q * kPickThreads + t;
        if (i >= n || !in[q] || !masses[i]) continue;
        const int idx = key_index(keys[i]);
        u64 b = 0;
        for (int j = 0; j < n; ++j) b += key_index(keys[j]) < idx ? masses[j] : 0;
        if (b <= place_at && place_at < b + masses[i]) pick = Pick{idx, key_value(keys[i])};
      }
    } else {
      // the bins before the cut's are in the chunks' sums; its kept words join theirs
      last = ~block_max<kPickThreads>(~last, tmp);
      if (t < C) chunks[t] = s.csum[t];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int i = q * kPickThreads + t;
        if (i < n && in[q] && masses[i]) {
          const int g = (key_index(keys[i]) + row.off) / RowView<DT>::E;
          // chunk c: the largest with chunk_at(c) <= g
          int c = (int)(((int64_t)g * C + C) / row.n);
          if (c >= C) c = C - 1;
          while (chunk_at(row.n, c, C) > g) --c;
          while (c + 1 < C && chunk_at(row.n, c + 1, C) <= g) ++c;
          atomicAdd(&chunks[c], masses[i]);
        }
      }
      __syncthreads();
      S = block_sum<kPickThreads>(t < C ? chunks[t] : 0, tmp);
      place_at = place(set.u, S);
      u64 in_chunk = place_at;
      const int c = pick_chunk(chunks, C, in_chunk, tmp, &at, &left);
      if (c >= 0)
        pick_in<DT>(row, mass, chunk_at(row.n, c, C), chunk_at(row.n, c + 1, C), in_chunk,
                    [&](u64 key, double w) {
                      return key == first || (w >= min_p && key >= last);
                    },
                    tmp, &pick);
    }
  } else if (hist) {
    // too many to list: the cut by radix over the row
    u64 upto = 0, cutk = 0;
    double total = (double)cut.total;
    if (set.by_k) {
      u64 k = 0, all = 0;
      for (int b = t; b < kBins; b += kPickThreads) k += s.count[b];
      all = block_sum<kPickThreads>(k, tmp);
      k = (u64)set.k < all ? (u64)set.k : all;
      cutk = select_key<DT>(row, mass, false, k, 0.0, upto, hm, hc, tmp, res);
      total = (double)upto;
    }
    if (set.by_p) cutk = select_key<DT>(row, mass, true, 0, (double)set.p * total, upto, hm, hc, tmp, res);
    if (t == 0) cutkey = cutk;
    __syncthreads();
    const u64 ck = cutkey;
    auto kept = [&](u64 key, double w) { return key == first || (w >= min_p && key >= ck); };
    u64 sum = 0;
    for (int g = t; g < row.n; g += kPickThreads) {
      float v[RowView<DT>::E];
      row.load(g, v);
#pragma unroll
      for (int e = 0; e < RowView<DT>::E; ++e) {
        if (!(v[e] > kNone)) continue;
        const double w = mass.w(v[e]);
        if (kept(order_key(v[e], row.first(g) + e), w)) sum += mass.of(w);
      }
    }
    S = block_sum<kPickThreads>(sum, tmp);
    place_at = place(set.u, S);
    pick_in<DT>(row, mass, 0, row.n, place_at, kept, tmp, &pick);
  } else {
    S = block_sum<kPickThreads>(t < C ? s.csum[t] : 0, tmp);
    place_at = place(set.u, S);
    u64 in_chunk = place_at;
    const int c = pick_chunk(s.csum, C, in_chunk, tmp, &at, &left);
    if (c >= 0)
      pick_in<DT>(row, mass, chunk_at(row.n, c, C), chunk_at(row.n, c + 1, C), in_chunk,
                  [&](u64 key, double w) { return key == first || w >= min_p; }, tmp, &pick);
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
    const dim3 grid((unsigned)C, (unsigned)a.R);
    auto go = [&](auto dtc) {
      constexpr int DT = decltype(dtc)::value;
      hipLaunchKernelGGL(sample_max_kernel<DT>, grid, dim3(kPassThreads), 0, st, a, ws, C);
      hipLaunchKernelGGL(sample_mass_kernel<DT>, grid, dim3(kPassThreads), 0, st, a, ws, C);
      hipLaunchKernelGGL(sample_list_kernel<DT>, grid, dim3(kPassThreads), 0, st, a, ws, C);
      hipLaunchKernelGGL(sample_pick_kernel<DT>, dim3((unsigned)a.R), dim3(kPickThreads), 0, st, a,
                         ws, C);
    };
    if (dtype == kBF16) go(std::integral_constant<int, kBF16>{});
    else if (dtype == kF16) go(std::integral_constant<int, kF16>{});
    else go(std::integral_constant<int, kF32>{});
    *nlaunch += 4;
  }
  return 0;
}

}  // namespace mq
