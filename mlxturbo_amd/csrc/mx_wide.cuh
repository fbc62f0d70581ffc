// Wide MXFP4 products: quantized_matmul (T) on the tile of mx_tile.cuh and qqmm (QQ:
// x packed into codes by mx_pack_kernel first) on that of mx_code.cuh.
#pragma once
#include "dense.cuh"
#include "mx_code.cuh"
#include "mx_tile.cuh"

namespace mq {

// x [M, K] -> codes and scales as the 4-bit tile takes them (mx_code.cuh): a
// thread takes 8 values, a group's four threads agree on its scale, groups past
// K are zero.  units = M * steps * 64.
template <int DT>
__global__ __launch_bounds__(256) void mx_pack_kernel(const uint16_t* __restrict__ x,
                                                      uint32_t* __restrict__ codes,
                                                      uint8_t* __restrict__ scales, int64_t units,
                                                      int G, int steps) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= units) return;
  const int64_t row = u / (steps * 64);
  const int k = (int)(u - row * (steps * 64)), g = k >> 2;    // 8-value unit, group of the row
  u32x4 v = (u32x4){0, 0, 0, 0};
  if (g < G) v = *reinterpret_cast<const u32x4*>(x + (row * G * 4 + k) * 8);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) top = mx_max2(top, v[j] & 0x7fff7fffu);
  const uint32_t e = mx_scale_byte<DT>(mx_quad_max(max(top & 0xffffu, top >> 16)));
  const uint32_t w = mx_code_word<DT>(v, mx_scale(e));
  // row m at m * steps * 64 words: the unit's own index
  codes[u] = e == 255 ? 0u : w;
  if ((k & 3) == 0)
    scales[(row * steps + (g >> 4)) * 16 + 4 * (g & 3) + ((g >> 2) & 3)] = (uint8_t)e;
}

// Tiles of rows that run side by side: six by five columns of weights move about as
// few bytes of x as of weights through an XCD's L2 (4096 rows, T, N=17408 K=5120:
// 522 us, all rows side by side 543).
constexpr int kMxGroupTiles = 6;

// Tile i: an XCD (i % 8) runs a contiguous range of the tiles in the order of
// groups of up to kMxGroupTiles tiles of rows, then weight columns (and shares of K), then
// the group's rows, so that the tiles that it runs at a time share both their x and
// their weights in its L2.
__device__ __forceinline__ bool mx_wide_tile(int i, int ncol, int mtiles, int& cz,
                                             int& mt) {
  int tile, one;
  if (!grouped_tile(i, ncol * mtiles, 1, tile, one)) return false;
  const int ng = (mtiles + kMxGroupTiles - 1) / kMxGroupTiles, h = (mtiles + ng - 1) / ng;
  const int g = tile / (h * ncol), rest = tile - g * h * ncol, rows = min(h, mtiles - g * h);
  cz = rest / rows;
  mt = g * h + rest - cz * rows;
  return true;
}

// A tile and a share z of the steps per workgroup (mx_wide_tile); where part is
// given the sums go to its float plane part[z].
template <int DT, bool QQ, int BM, bool TAIL>
__global__ __launch_bounds__(256, BM <= 64 && !QQ ? 2 : 1) void mx_wide_kernel(
    const void* __restrict__ x, const uint8_t* __restrict__ xscales,
    const uint32_t* __restrict__ w, const uint8_t* __restrict__ scales,
    uint16_t* __restrict__ out, float* __restrict__ part, int M, int N, int G, int splits) {
  using Sh = MxTileShape<BM>;
  using Shc = MxCodeShape<BM>;
  __shared__ __align__(16) unsigned char A0[QQ ? Shc::kHalf : Sh::kStage];
  __shared__ __align__(16) unsigned char A1[QQ ? Shc::kHalf : Sh::kStage];
  __shared__ __align__(16) unsigned char A2[QQ ? Shc::kScales : Sh::kStages > 2 ? Sh::kStage : 16];
  __shared__ __align__(16) unsigned char A3[!QQ && Sh::kStages > 2 ? Sh::kStage : 16];
  int cz, mt;
  if (!mx_wide_tile(blockIdx.x, (N + 255) / 256 * splits, (M + BM - 1) / BM, cz, mt)) return;
  const int col = cz / splits, z = cz - col * splits;
  const int m0 = mt * BM, n0 = col * 256;
  const int mrows = min(BM, M - m0), ncols = min(256, N - n0);
  const int steps = QQ ? (G + 15) / 16 : (G + 3) / 4;
  constexpr int kUnit = QQ || TAIL ? 1 : Sh::kStages;
  const int nu = steps / kUnit;
  const int kt0 = kUnit * (int)((int64_t)nu * z / splits);
  const int kt1 = kUnit * (int)((int64_t)nu * (z + 1) / splits);
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t rowb = QQ ? (uint32_t)steps * 256u : (uint32_t)G * 64u;
  const auto xr = wide_rsrc((const unsigned char*)x + (int64_t)m0 * rowb, (int64_t)mrows * rowb);
  const auto xs = wide_rsrc(QQ ? xscales + (int64_t)m0 * steps * 16 : nullptr,
                            QQ ? (int64_t)mrows * steps * 16 : 0);
  const bool vec = N % 4 == 0 && (part || (uintptr_t)out % 8 == 0);
  // the four sums v of x row m and weight rows n ..
  auto put = [&](int m, int n, const f32x4& v) {
    if (m >= mrows) return;
    if (part) {
      float* o = part + ((int64_t)z * M + m0 + m) * N + n0 + n;
      if (vec) {
        if (n < ncols) *reinterpret_cast<f32x4*>(o) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < ncols) o[e] = v[e];
      }
      return;
    }
    uint16_t* o = out + (int64_t)(m0 + m) * N + n0 + n;
    if (vec) {
      if (n < ncols)
        *reinterpret_cast<u32x2*>(o) =
            (u32x2){T16<DT>::pack2(v[0], v[1]), T16<DT>::pack2(v[2], v[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < ncols) o[e] = T16<DT>::round1(v[e]);
    }
  };
  const uint32_t* wt = w + (int64_t)n0 * G * 4;
  const uint8_t* st = scales + (int64_t)n0 * G;
  if constexpr (QQ)
    mx_code_tile<BM, TAIL>(
        xr, xs, wt, st, ncols, G, steps, kt0, kt1 - kt0,
        [&](int i, int j, const f32x4& v) {
          put(BM / 2 * (wave & 1) + 16 * i + r, 128 * (wave >> 1) + 16 * j + 4 * c, v);
        },
        A0, A1, A2);
  else
    mx_tile<DT, BM, TAIL>(
        xr, [&](int i) { return i < mrows ? (uint32_t)i * rowb : 0x80000000u; }, wt, st, ncols, G, kt0, kt1 - kt0,
        [&](int i, int j, const f32x4& v) {
          put(16 * i + r, 64 * wave + 16 * j + 4 * c, v);
        },
        A0, A1, A2, A3);
}

template <int DT, bool QQ, int BM>
inline int mx_wide_launch_bm(const void* x, const uint8_t* xs, const uint32_t* w,
                             const uint8_t* s, void* out, int64_t M, int64_t N, int64_t K,
                             int splits, float* part, hipStream_t st) {
  const int64_t G = K / kMxGroup, tiles = (N + 255) / 256 * ((M + BM - 1) / BM) * splits;
  if (!mx_grid_ok((tiles + 7) / 8 * 8, 256)) return kStatusUnsupported;
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8));
  auto go = [&](auto tail) {
    hipLaunchKernelGGL((mx_wide_kernel<DT, QQ, BM, decltype(tail)::value>), grid, dim3(256), 0,
                       st, x, xs, w, s, (uint16_t*)out, part, (int)M, (int)N, (int)G, splits);
  };
  if (G % 16) go(std::true_type{});
  else go(std::false_type{});
  if (splits > 1) {
    const int64_t MN = M * N;
    const dim3 rg((unsigned)((MN + 1023) / 1024));
    if (MN % 4 == 0 && (uintptr_t)out % 8 == 0)
      hipLaunchKernelGGL((wide_reduce_kernel<DT, true>), rg, dim3(256), 0, st, part,
                         (uint16_t*)out, MN, splits);
    else
      hipLaunchKernelGGL((wide_reduce_kernel<DT, false>), rg, dim3(256), 0, st, part,
                         (uint16_t*)out, MN, splits);
  }
  return 0;
}

// (x packed into ws: mx_pack_bytes)
template <int DT>
inline void mx_pack_launch(const void* x, void* ws, int64_t M, int64_t K, hipStream_t st) {
  const int64_t steps = (K + 511) / 512, units = M * steps * 64;
  uint8_t* xs = static_cast<uint8_t*>(ws) + M * steps * kMxStepBytes;
  hipLaunchKernelGGL(mx_pack_kernel<DT>, dim3((unsigned)((units + 255) / 256)), dim3(256), 0, st,
                     (const uint16_t*)x, (uint32_t*)ws, xs, units, (int)(K / kMxGroup),
                     (int)steps);
}

template <int DT, bool QQ>
int MxWideLaunch<DT, QQ>::run(const void* x, const uint32_t* w, const uint8_t* s, void* out,
                              int64_t M, int64_t N, int64_t K, void* ws, size_t ws_bytes,
                              hipStream_t st, int* nlaunch) {
  if (!mx_wide_fits(M, N, K)) return kStatusUnsupported;
  const int cus = device_cu_count();
  MxWidePlan plan = mx_wide_plan(M, N, K, QQ, cus);
  if (ws_bytes < mx_wide_workspace_bytes(plan, M, N, K, QQ)) {
    plan = mx_wide_plan(M, N, K, QQ, cus, 1);
    if (ws_bytes < mx_wide_workspace_bytes(plan, M, N, K, QQ)) return kStatusUnsupported;
  }
  const uint8_t* xs = nullptr;
  float* part = static_cast<float*>(ws);
  if (QQ) {
    mx_pack_launch<DT>(x, ws, M, K, st);
    xs = static_cast<uint8_t*>(ws) + M * ((K + 511) / 512) * kMxStepBytes;
    x = ws;
    part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) +
                                    ((mx_pack_bytes(M, K) + 255) & ~(size_t)255));
    *nlaunch += 1;
  }
  if (plan.splits == 1) part = nullptr;
  *nlaunch += plan.splits > 1 ? 2 : 1;
  switch (plan.bm) {
    case 64:
      return mx_wide_launch_bm<DT, QQ, 64>(x, xs, w, s, out, M, N, K, plan.splits, part, st);
    case 128:
      return mx_wide_launch_bm<DT, QQ, 128>(x, xs, w, s, out, M, N, K, plan.splits, part, st);
    default:
      return mx_wide_launch_bm<DT, QQ, 192>(x, xs, w, s, out, M, N, K, plan.splits, part, st);
  }
}

}  // namespace mq
