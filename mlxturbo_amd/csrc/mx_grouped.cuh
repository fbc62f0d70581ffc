// gather_qmm of many pairs on the MXFP4 tile (mx_tile.cuh): a workgroup runs a
// segment of up to BM rows of one expert (the prep kernels' tables, prep.hip)
// times 256 weight rows.
//
// x rows are gathered by the tile's LDS-form loads themselves (each lane's row
// offset is looked up after the first weights are issued) and output rows
// scattered back to pair order.  Bound by the weights: experts with few rows
// make a tile mostly weights, whole lines of 16 rows per two loads, two to three
// steps ahead, two workgroups per CU; a tile is as tall as its rows need (16, 32
// or 64: with 64 for all, 128 experts of N=768 K=2048 at 19 rows each took 46
// us).
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
  mx_tile<DT, false, BM, TAIL>(
      xr,
      [&](int i) {
        if (i >= rows) return 0x80000000u;      // zeros, no memory access
        const int q = Mi == 1 ? i : i / Mi;
        return (uint32_t)(((int64_t)x_batch(lhs, lds.pair[q], P, B) * Mi + i - q * Mi) * G * 64);
      },
      xr, [](int) { return 0u; }, w + row0 * G * 4, scales + row0 * G, ncols, G, 0, (G + 3) / 4,
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

// Over the prep kernels' tables.  Grid: BM = 64, the tables of
// launch_thin_tables: class 1 (segments of up to 2 (64 / Mi) pairs, run as two
// adjacent tiles) in the first 8 q1 workgroups (q1 = its tiles / 8, rounded up),
// then class 0; else class 0 alone, segments of up to BM / Mi pairs.  Tiles
// placed by grouped_tile.  B * Mi * K * 2 < 2^31.
template <int DT, int BM, bool TAIL>
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
  const int32_t* hdr = ws + gather_ws_header(P);
  const int ncol = (N + 255) / 256;
  int bi = blockIdx.x, cls = 0;
  if constexpr (BM == 64) {
    const int q1 = (2 * (hdr[2] - hdr[1]) * ncol + 7) / 8;
    if (bi < 8 * q1) cls = 1;
    else bi -= 8 * q1;
  }
  int seg, col;
  if (!grouped_tile(bi, (hdr[3 - cls] - hdr[2 - cls]) * (cls + 1), ncol, seg, col)) return;
  const int pofs = cls ? (seg & 1) * (BM / Mi) : 0;
  seg = (cls ? seg >> 1 : seg) + hdr[2 - cls];
  const int32_t* perm = ws + 1;
  const int st0 = perm[P + seg] + pofs, len = min(perm[2 * P + seg] - pofs, BM / Mi);
  if (len <= 0) return;                         // an empty half of a segment
  const int e = __builtin_amdgcn_readfirstlane(perm[3 * P + seg]);
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

// Without tables, for up to kMxListP pairs: a workgroup reads all expert indices
// (16 per thread) and lists its expert's pairs in pair order itself, one launch
// instead of three (the tables of 2408 pairs take 17 us).  Workgroup (z, expert,
// column) runs segments z, z + Z, ... of 64 / Mi pairs; "expert" E are the pairs
// that get zeros.  Grid: per z, all experts' first segments first, (E + 1) * ncol
// tiles by grouped_tile.
constexpr int kMxListP = 4096;

template <int DT, bool TAIL>
__global__ __launch_bounds__(256, 2) void mx_listed_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ w,
    const uint8_t* __restrict__ scales, const int32_t* __restrict__ lhs,
    const int32_t* __restrict__ rhs, uint16_t* __restrict__ out, int P, int B, int Mi, int N,
    int G, int E, int Z) {
  using Sh = MxTileShape<64>;
  __shared__ __align__(16) unsigned char A0[Sh::kStage];
  __shared__ __align__(16) unsigned char A1[Sh::kStage];
  __shared__ __align__(16) unsigned char A2[Sh::kStage];
  __shared__ __align__(16) unsigned char A3[Sh::kStage];
  __shared__ int s_pair[64];
  __shared__ int s_wave[4];
  const int ncol = (N + 255) / 256, t = threadIdx.x, lane = t & 63;
  const int nz = ((E + 1) * ncol + 7) / 8 * 8, z = blockIdx.x / nz;
  int e, col;
  if (!grouped_tile(blockIdx.x - z * nz, E + 1, ncol, e, col)) return;
  constexpr int PER = kMxListP / 256;
  const int per = (P + 255) >> 8, p0 = t * per;  // this thread's pairs
  uint32_t mask = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int p = p0 + i;
    if (i < per && p < P) {
      int k = rhs[p];
      const int b = x_batch(lhs, p, P, B);
      k = k >= 0 && k < E && b >= 0 && b < B ? k : E;
      mask |= (uint32_t)(k == e) << i;
    }
  }
  // exclusive prefix of the threads' counts
  const int cnt = __popc(mask);
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
  const int R = 64 / Mi;
  const MxGroupedLds<64> lds{{A0, A1, A2, A3}, s_pair};
  for (int s0 = z * R; s0 < total; s0 += Z * R) {
    __syncthreads();                            // the last segment's pairs are read
    int rank = before;
    for (uint32_t m = mask; m; m &= m - 1, ++rank)
      if (rank >= s0 && rank < s0 + R) s_pair[rank - s0] = p0 + __builtin_ctz(m);
    __syncthreads();
    const int rows = min(R, total - s0) * Mi;
    if (e >= E) mx_zero_rows(s_pair, out, rows, col, Mi, N);
    else mx_thin_tile<DT, TAIL>(lds, x, w, scales, lhs, out, rows, e, col, P, B, Mi, N, G);
  }
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
  const int64_t ncol = (N + 255) / 256, R = 192 / M;
  if (!tall && P <= kMxListP) {
    // an expert's segments spread over up to 4 workgroups
    const int64_t Z = P * M <= 64 ? 1 : 4, ntile = ((E + 1) * ncol + 7) / 8 * 8 * Z;
    if (ntile > INT32_MAX) return kStatusUnsupported;
    auto go = [&](auto tail) {
      hipLaunchKernelGGL((mx_listed_kernel<DT, decltype(tail)::value>), dim3((unsigned)ntile),
                         dim3(256), 0, st, (const uint16_t*)x, w, s, lhs, rhs, (uint16_t*)out,
                         (int)P, (int)B, (int)M, (int)N, (int)G, (int)E, (int)Z);
    };
    if (G % 16) go(std::true_type{});
    else go(std::false_type{});
    *nlaunch += 1;
    return 0;
  }
  const int64_t nwg =
      tall ? (class_seg_bound(P, R, 0, E) * ncol + 7) / 8 * 8 : thin_grid(P, M, N, E, false);
  if (nwg > INT32_MAX) return kStatusUnsupported;
  if (int rc = tall ? launch_prep(rhs, lhs, P, E, B, (int)R, ws, st)
                    : launch_thin_tables(rhs, lhs, P, E, B, M, ws, st))
    return rc;
  *nlaunch += kPrepLaunches + 1;
  auto go = [&](auto bm, auto tail) {
    hipLaunchKernelGGL((mx_grouped_kernel<DT, decltype(bm)::value, decltype(tail)::value>),
                       dim3((unsigned)nwg), dim3(256), 0, st, (const uint16_t*)x, w, s, lhs,
                       (uint16_t*)out, (const int32_t*)ws, (int)P, (int)B, (int)M, (int)N, (int)G,
                       (int)E);
  };
  using Tall = std::integral_constant<int, 192>;
  using Thin = std::integral_constant<int, 64>;
  if (tall) {
    if (G % 16) go(Tall{}, std::true_type{});
    else go(Tall{}, std::false_type{});
  } else {
    if (G % 16) go(Thin{}, std::true_type{});
    else go(Thin{}, std::false_type{});
  }
  return 0;
}

}  // namespace mq
