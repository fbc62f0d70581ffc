// gather_qmm of many pairs on the MXFP4 tile (mx_tile.cuh): a workgroup runs a
// segment of up to BM rows of one expert (the prep kernels' tables, prep.hip)
// times 256 weight rows.
//
// x rows are gathered by the tile's LDS-form loads themselves (each lane's row
// offset is looked up after the first weights are issued) and output rows
// scattered back to pair order.  Bound by the weights: experts with few rows
// make a tile mostly weights, 64 contiguous bytes of 16 rows per load, two steps
// ahead, two workgroups per CU.
#pragma once
#include "mx_tile.cuh"

namespace mq {

// Grid: BM = 64, the tables of launch_thin_tables: class 1 (segments of up to 2
// (64 / Mi) pairs, run as two adjacent tiles) in the first 8 q1 workgroups (q1 =
// its tiles / 8, rounded up), then class 0; else class 0 alone, segments of up to
// BM / Mi pairs.  Tiles placed by grouped_tile.  Segments of pairs whose expert
// or x batch does not exist write zeros.  B * Mi * K * 2 < 2^31.
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
  __shared__ int s_orow[BM];
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
  const int rows = len * Mi;                    // <= BM
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n0 = col * 256, ncols = min(256, N - n0);
  // tile row r: row r % Mi of pair perm[st0 + r / Mi]
  if (t < BM) {
    const int q = Mi == 1 ? t : t / Mi;
    s_orow[t] = t < rows ? perm[st0 + q] * Mi + t - q * Mi : -1;
  }
  if (e >= E) {
    __syncthreads();
    for (int i = t; i < rows * ncols; i += 256) {
      const int a = i / ncols;
      out[(int64_t)s_orow[a] * N + n0 + i - a * ncols] = 0;
    }
    return;
  }
  const auto xr = wide_rsrc(x, (int64_t)B * Mi * G * 64);
  const int64_t row0 = (int64_t)e * N + n0;
  const bool vec = N % 4 == 0 && (uintptr_t)out % 8 == 0;
  mx_tile<DT, false, BM, TAIL>(
      xr,
      [&](int i) {
        if (i >= rows) return 0x80000000u;      // zeros, no memory access
        const int q = Mi == 1 ? i : i / Mi, p = perm[st0 + q];
        return (uint32_t)(((int64_t)x_batch(lhs, p, P, B) * Mi + i - q * Mi) * G * 64);
      },
      xr, [](int) { return 0u; }, w + row0 * G * 4, scales + row0 * G, ncols, G, 0, (G + 3) / 4,
      [&](int i, int j, const f32x4& v) {
        const int o = s_orow[16 * i + r], n = 64 * wave + 16 * j + 4 * c;
        if (o < 0) return;
        uint16_t* d = out + (int64_t)o * N + n0 + n;
        if (vec) {
          if (n < ncols)
            *reinterpret_cast<u32x2*>(d) =
                (u32x2){T16<DT>::pack2(v[0], v[1]), T16<DT>::pack2(v[2], v[3])};
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (n + q < ncols) d[q] = T16<DT>::round1(v[q]);
        }
      },
      A0, A1, A2, A3);
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
    if (G % 4) go(Tall{}, std::true_type{});
    else go(Tall{}, std::false_type{});
  } else {
    if (G % 4) go(Thin{}, std::true_type{});
    else go(Thin{}, std::false_type{});
  }
  return 0;
}

}  // namespace mq
