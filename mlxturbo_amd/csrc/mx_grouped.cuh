// gather_qmm of many pairs on the MXFP4 tile (mx_tile.cuh): a workgroup runs a
// segment of up to BM rows of one expert times 256 weight rows.
//
// x rows are gathered by the tile's LDS-form loads themselves (each lane's row
// offset is looked up after the first weights are issued) and output rows
// scattered back to pair order.  Bound by the weights: experts with few rows
// make a tile mostly weights, whole lines of 16 rows per two loads, four steps
// ahead, two workgroups per CU; a tile is as tall as its rows need (16, 32 or
// 64).  2408 pairs over 128 experts of N=768 K=2048: 32 us, 3.4 TB/s of weights;
// 16384 over 512 of N=512 K=2048: 91 us, 3.1 TB/s; K that is not whole 512s (N=2048
// K=768, 2408 pairs over 128): 41 us, 2.6 TB/s.
#pragma once
#include "mx_tile.cuh"

namespace mq {

template <int BM> struct MxGroupedLds {
  unsigned char* A[4];
  const int* pair;                              // the tile's pairs
};

// One tile: rows (<= BM) of the pairs in lds.pair (Mi rows each) of expert e
// times weight rows [256 col, +256).  Every thread of the workgroup calls.
template <int DT, int BM, bool TAIL, int LBM>
__device__ __forceinline__ void mx_grouped_tile(const MxGroupedLds<LBM>& lds,
                                                const uint16_t* __restrict__ x,
                                                const uint32_t* __restrict__ w,
                                                const uint8_t* __restrict__ scales,
                                                const int32_t* __restrict__ lhs,
                                                uint16_t* __restrict__ out, int rows, int e,
                                                int col, int P, int B, int Mi, int N, int G) {
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = col * 256, ncols = min(256, N - n0);
  const auto xr = wide_rsrc(x, (int64_t)B * Mi * G * 64);
  const int64_t row0 = (int64_t)e * N + n0;
  const bool vec = N % 4 == 0 && (uintptr_t)out % 8 == 0;
  mx_tile<DT, BM, TAIL>(
      xr,
      [&](int i) {
        if (i >= rows) return 0x80000000u;      // zeros, no memory access
        const int q = Mi == 1 ? i : i / Mi;
        return (uint32_t)(((int64_t)x_batch(lhs, lds.pair[q], P, B) * Mi + i - q * Mi) * G * 64);
      },
      w + row0 * G * 4, scales + row0 * G, ncols, G, 0, (G + 3) / 4,
      [&](int i, int j, const f32x4& v) {
        const int m = 16 * i + r, n = 64 * wave + 16 * j + 4 * c;
        if (m >= rows) return;
        const int q = Mi == 1 ? m : m / Mi;
        uint16_t* d = out + ((int64_t)lds.pair[q] * Mi + m - q * Mi) * N + n0 + n;
        if (vec) {
          if (n < ncols)
            *reinterpret_cast<u32x2*>(d) =
                (u32x2){T16<DT>::pack2(v[0], v[1]), T16<DT>::pack2(v[2], v[3])};
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n + k < ncols) d[k] = T16<DT>::round1(v[k]);
        }
      },
      lds.A[0], lds.A[1], lds.A[2], lds.A[3]);
}

// The tile of least height, 16, 32 or 64, that holds the rows.
template <int DT, bool TAIL>
__device__ __forceinline__ void mx_thin_tile(const MxGroupedLds<64>& lds,
                                             const uint16_t* __restrict__ x,
                                             const uint32_t* __restrict__ w,
                                             const uint8_t* __restrict__ scales,
                                             const int32_t* __restrict__ lhs,
                                             uint16_t* __restrict__ out, int rows, int e, int col,
                                             int P, int B, int Mi, int N, int G) {
  if (rows <= 16)
    mx_grouped_tile<DT, 16, TAIL>(lds, x, w, scales, lhs, out, rows, e, col, P, B, Mi, N, G);
  else if (rows <= 32)
    mx_grouped_tile<DT, 32, TAIL>(lds, x, w, scales, lhs, out, rows, e, col, P, B, Mi, N, G);
  else
    mx_grouped_tile<DT, 64, TAIL>(lds, x, w, scales, lhs, out, rows, e, col, P, B, Mi, N, G);
}

// Zero rows of the tile's pairs (no such expert or x batch).
__device__ __forceinline__ void mx_zero_rows(const int* pair, uint16_t* __restrict__ out, int rows,
                                             int col, int Mi, int N) {
  const int n0 = col * 256, ncols = min(256, N - n0);
  for (int i = threadIdx.x; i < rows * ncols; i += 256) {
    const int a = i / ncols, q = a / Mi;
    out[((int64_t)pair[q] * Mi + a - q * Mi) * N + n0 + i - a * ncols] = 0;
  }
}

// Pairs sorted by expert, up to kMxSortP of them, without a serial pass: workgroup
// e of E + 1 reads all keys (the expert, or E where it or the x batch is out of
// range), counts those below e, which is where e's pairs begin, and writes its
// own: perm, then starts[E + 2].  Bound by its one round of loads and the launch
// (16384 pairs, 512 experts: 8.7 us; the tables of launch_prep 19).
constexpr int64_t kMxSortP = 32768;
__host__ __device__ inline size_t mx_sort_starts(int64_t P) { return ((size_t)P + 3) & ~(size_t)3; }

template <int W>   // 64-bit masks per thread: up to W * 16384 pairs
__global__ __launch_bounds__(256) void mx_sort_kernel(const int32_t* __restrict__ rhs,
                                                      const int32_t* __restrict__ lhs, int P,
                                                      int B, int E, int32_t* __restrict__ ws) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  auto load_i4 = [](__amdgpu_buffer_rsrc_t r, int p) {       // zeros past the end
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, 4 * p, 0, 0));
  };
  __shared__ int s_eq[4], s_lt[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, e = blockIdx.x;
  // step i of a wave: 256 pairs, four per lane
  const int steps = (P + 1023) >> 10, p0 = (wave * steps << 8) + 4 * lane;
  const auto rk = wide_rsrc(rhs, (int64_t)P * 4), rb = wide_rsrc(lhs, lhs ? (int64_t)P * 4 : 0);
  uint64_t mask[W] = {};
  int lt = 0;
#pragma unroll
  for (int m = 0; m < 2 * W; ++m) {              // eight steps' loads in flight
    if (8 * m >= steps) break;
    i32x4 k[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = load_i4(rk, p0 + ((8 * m + i) << 8));
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = lhs ? load_i4(rb, p0 + ((8 * m + i) << 8)) : (i32x4){};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // steps past the wave's own are other waves' pairs
      const int left = 8 * m + i < steps ? P - p0 - ((8 * m + i) << 8) : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key =
            (uint32_t)k[i][j] < (uint32_t)E && (uint32_t)b[i][j] < (uint32_t)B && j < left
                ? k[i][j]
                : E;
        lt += key < e;
        mask[m / 2] |= (uint64_t)(key == e && j < left) << (4 * (8 * (m & 1) + i) + j);
      }
    }
  }
  int cnt = 0;
#pragma unroll
  for (int m = 0; m < W; ++m) cnt += __popcll(mask[m]);
  int incl = cnt;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(incl, d), l = __shfl_xor(lt, d);
    if (lane >= d) incl += o;
    lt += l;
  }
  if (lane == 63) {
    s_eq[wave] = incl;
    s_lt[wave] = lt;
  }
  __syncthreads();
  const int start = s_lt[0] + s_lt[1] + s_lt[2] + s_lt[3];
  int at = start + incl - cnt;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < wave) at += s_eq[i];
#pragma unroll
  for (int m = 0; m < W; ++m)
    for (uint64_t b = mask[m]; b; b &= b - 1) {
      const int i = __builtin_ctzll(b);
      ws[at++] = p0 + ((16 * m + (i >> 2)) << 8) + (i & 3);
    }
  if (t == 0) {
    ws[mx_sort_starts(P) + e] = start;
    if (e == E) ws[mx_sort_starts(P) + E + 1] = P;
  }
}

// Segments of up to R = BM / Mi pairs times 256 columns, placed by grouped_tile.
// SORTED: ws as mx_sort_kernel writes it, and every workgroup finds its segment
// itself by a scan of the experts' segment counts; else launch_prep's tables of
// one class.  BM = 64: a tile as tall as its rows need.  B * Mi * K * 2 < 2^31.
template <int DT, int BM, bool TAIL, bool SORTED>
__global__ __launch_bounds__(256, BM <= 64 ? 2 : 1) void mx_grouped_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ w,
    const uint8_t* __restrict__ scales, const int32_t* __restrict__ lhs,
    uint16_t* __restrict__ out, const int32_t* __restrict__ ws, int P, int B, int Mi, int N, int G,
    int E) {
  using Sh = MxTileShape<BM>;
  __shared__ __align__(16) unsigned char A0[Sh::kStage];
  __shared__ __align__(16) unsigned char A1[Sh::kStage];
  __shared__ __align__(16) unsigned char A2[Sh::kStages > 2 ? Sh::kStage : 16];
  __shared__ __align__(16) unsigned char A3[Sh::kStages > 2 ? Sh::kStage : 16];
  __shared__ int s_pair[BM];
  const int ncol = (N + 255) / 256, R = BM / Mi;
  int seg, col, e, st0, len;
  const int32_t* perm = ws;
  if constexpr (SORTED) {
    __shared__ int s_wave[4], s_seg[3];
    const int32_t* starts = ws + mx_sort_starts(P);
    constexpr int PER = (kGatherPrepMaxE + 1 + 255) / 256;
    const int t = threadIdx.x, lane = t & 63, per = (E + 256) / 256;   // of E + 1 keys
    int s[PER + 1], cnt = 0;
#pragma unroll
    for (int i = 0; i <= PER; ++i) s[i] = i <= per ? starts[min(t * per + i, E + 1)] : 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < per) cnt += (s[i + 1] - s[i] + R - 1) / R;
    int incl = cnt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    if (lane == 63) s_wave[t >> 6] = incl;
    __syncthreads();
    int before = incl - cnt, total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < (t >> 6)) before += s_wave[i];
      total += s_wave[i];
    }
    total = __builtin_amdgcn_readfirstlane(total);
    if (!grouped_tile(blockIdx.x, total, ncol, seg, col)) return;
    if (seg >= before && seg < before + cnt) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < per) {
          const int n = (s[i + 1] - s[i] + R - 1) / R;
          if (seg >= before && seg < before + n) {
            s_seg[0] = t * per + i;
            s_seg[1] = s[i] + (seg - before) * R;
            s_seg[2] = min(R, s[i + 1] - s_seg[1]);
          }
          before += n;
        }
    }
    __syncthreads();
    e = __builtin_amdgcn_readfirstlane(s_seg[0]);
    st0 = s_seg[1];
    len = __builtin_amdgcn_readfirstlane(s_seg[2]);
  } else {
    if (!grouped_tile(blockIdx.x, ws[0], ncol, seg, col)) return;
    perm = ws + 1;
    st0 = perm[P + seg];
    len = perm[2 * P + seg];
    e = __builtin_amdgcn_readfirstlane(perm[3 * P + seg]);
  }
  if ((int)threadIdx.x < len) s_pair[threadIdx.x] = perm[st0 + threadIdx.x];
  __syncthreads();
  if (e >= E) {
    mx_zero_rows(s_pair, out, len * Mi, col, Mi, N);
    return;
  }
  const MxGroupedLds<BM> lds{{A0, A1, A2, A3}, s_pair};
  if constexpr (BM == 64)
    mx_thin_tile<DT, TAIL>(lds, x, w, scales, lhs, out, len * Mi, e, col, P, B, Mi, N, G);
  else
    mx_grouped_tile<DT, BM, TAIL>(lds, x, w, scales, lhs, out, len * Mi, e, col, P, B, Mi, N, G);
}

template <int DT>
int MxGroupedLaunch<DT>::run(const void* x, const uint32_t* w, const uint8_t* s,
                             const int32_t* lhs, const int32_t* rhs, void* out, int64_t P,
                             int64_t B, int64_t M, int64_t N, int64_t K, int64_t E, void* ws,
                             hipStream_t st, int* nlaunch) {
  if (B * M * K * 2 >= ((int64_t)1 << 31) || K >= ((int64_t)1 << 21) || E > kGatherPrepMaxE)
    return kStatusUnsupported;
  const int64_t G = K / kMxGroup;
  // 96 rows per active expert and more: tall tiles read an expert's weights
  // once per 192 rows
  const bool tall = P * M / (P < E ? P : E) >= 96;
  const int64_t ncol = (N + 255) / 256, R = (tall ? 192 : 64) / M;
  const int64_t nwg = (class_seg_bound(P, R, 0, E) * ncol + 7) / 8 * 8;
  if (!mx_grid_ok(nwg, 256)) return kStatusUnsupported;
  const bool sorted = P <= kMxSortP;
  if (!sorted) {
    if (int rc = launch_prep(rhs, lhs, P, E, B, (int)R, ws, st)) return rc;
    *nlaunch += kPrepLaunches + 1;
  } else {
    auto sort = P <= kMxSortP / 2 ? mx_sort_kernel<1> : mx_sort_kernel<2>;
    hipLaunchKernelGGL(sort, dim3((unsigned)E + 1), dim3(256), 0, st, rhs, lhs, (int)P, (int)B,
                       (int)E, (int32_t*)ws);
    *nlaunch += 2;
  }
  auto go = [&](auto bm, auto tail, auto srt) {
    hipLaunchKernelGGL(
        (mx_grouped_kernel<DT, decltype(bm)::value, decltype(tail)::value, decltype(srt)::value>),
        dim3((unsigned)nwg), dim3(256), 0, st, (const uint16_t*)x, w, s, lhs, (uint16_t*)out,
        (const int32_t*)ws, (int)P, (int)B, (int)M, (int)N, (int)G, (int)E);
  };
  auto tails = [&](auto bm, auto srt) {
    if (G % 16) go(bm, std::true_type{}, srt);
    else go(bm, std::false_type{}, srt);
  };
  auto heights = [&](auto srt) {
    if (tall) tails(std::integral_constant<int, 192>{}, srt);
    else tails(std::integral_constant<int, 64>{}, srt);
  };
  if (sorted) heights(std::true_type{});
  else heights(std::false_type{});
  return 0;
}

}  // namespace mq
