// Launchers of the MXFP4 kernels, called by the C ABI (abi.hip); each enqueues
// on the given stream and returns 0, a HIP error or kStatusUnsupported.
#pragma once
#include "launch.h"

namespace mq {

constexpr int kMxGroup = 32;                    // codes per scale

// (wq, scales) = the MXFP4 codes of w [N, K] (any of the three dtypes), and
// back (mx_formats.hip).
int launch_mx_quantize(const void* w, uint32_t* wq, uint8_t* scales, int64_t N, int64_t K,
                       int dtype, hipStream_t st);
int launch_mx_dequantize(const uint32_t* wq, const uint8_t* scales, void* out, int64_t N,
                         int64_t K, int dtype, hipStream_t st);

// out [M, N] = x [M, K] . deq(w)^T on the skinny kernel (mx_skinny.cuh), 16 rows
// at a time; QQ: x brought into MXFP4 first.  Any M; *nlaunch counts the kernels enqueued.
template <int DT, bool QQ>
struct MxSkinnyLaunch {
  static int run(const void* x, const uint32_t* w, const uint8_t* s, void* out, int64_t M,
                 int64_t N, int64_t K, hipStream_t st, int* nlaunch);
};

// The same on the MFMA tile (mx_wide.cuh); ws of ws_bytes holds
// mx_wide_workspace_bytes of the plan, or of the plan without K splits.
template <int DT, bool QQ>
struct MxWideLaunch {
  static int run(const void* x, const uint32_t* w, const uint8_t* s, void* out, int64_t M,
                 int64_t N, int64_t K, void* ws, size_t ws_bytes, hipStream_t st, int* nlaunch);
};

// ---- the wide tile's plan ----------------------------------------------------

constexpr int kMxStepBytes = 256;               // of codes of an x row per 512 of K

// Bytes of x packed for the 4-bit tile: codes of whole steps, then scales.
inline size_t mx_pack_bytes(int64_t M, int64_t K) {
  return (size_t)(M * ((K + 511) / 512)) * (kMxStepBytes + 16);
}

// A tile's x rows and weight rows have to fit 31-bit buffer ranges, the grids (the
// packing of x has 64 threads per row and 512 codes) 32-bit thread counts.
inline bool mx_wide_fits(int64_t M, int64_t N, int64_t K) {
  return K < ((int64_t)1 << 21) && (M + 63) / 64 * ((N + 255) / 256) < ((int64_t)1 << 24) - 8 &&
         M * ((K + 511) / 512) < ((int64_t)1 << 26) && M * N < ((int64_t)1 << 40);
}

// Tile height and K split of least modelled cost, fitted to 20 to 2048 rows at
// N x K = 5120 x 17408, 17408 x 5120 and 4096 x 4096 (whole 512s; the same plan
// serves other K, whose steps take somewhat longer), splits 1 to 12, weights from
// memory (chosen tiles within 1%, QQ 2.5%, of the best measured, on average):
//  * a round of a tile per CU takes c0 and t per step (two 64-row tiles of T side by
//    side on a CU take as long as in turn), in more than one round at least tp per
//    step and tile of a CU;
//  * K splits sum into float planes that a second kernel adds, c1 and (8 S + 2) M N
//    bytes at bw.
struct MxWidePlan {
  int bm = 192, splits = 1;
  double cost_us = 0.0;
};

inline MxWidePlan mx_wide_plan(int64_t M, int64_t N, int64_t K, bool qq, int cus,
                               int max_splits = 16) {
  const int bms[3] = {192, 128, 64};
  const double us[2][3] = {{1.62, 1.3, 0.8}, {2.4, 2.1, 1.53}};   // t: of 128, QQ 512 codes
  const double held[2][3] = {{1.94, 1.04, 0.81}, {3.7, 2.06, 2.33}};     // tp
  const double c0 = qq ? 4.8 : 3.1, c1 = qq ? 4.0 : 2.7, bw = qq ? 5.5e6 : 5.2e6;
  const int64_t nk = qq ? (K + 511) / 512 : (K + 127) / 128, cols = (N + 255) / 256;
  const int64_t unit = qq || K % 512 ? 1 : 4;   // steps that a split takes or leaves
  MxWidePlan best;
  for (int sp = 1; sp <= max_splits; ++sp) {
    const int64_t steps = (nk / unit + sp - 1) / sp * unit;
    if (sp > 1 && (steps < 4 || sp > nk / unit)) break;
    for (int i = 0; i < 3; ++i) {
      const int64_t tiles = cols * ((M + bms[i] - 1) / bms[i]) * sp;
      const double round = c0 + us[qq][i] * (double)steps;
      double cost = (double)((tiles + cus - 1) / cus) * round;
      const double many = c0 + (double)tiles / cus * held[qq][i] * (double)steps;
      if (tiles > cus && many > cost) cost = many;
      if (sp > 1) cost += c1 + (8.0 * sp + 2.0) * (double)M * (double)N / bw;
      if (best.cost_us == 0.0 || cost < best.cost_us) {
        best.bm = bms[i];
        best.splits = sp;
        best.cost_us = cost;
      }
    }
  }
  return best;
}

inline size_t mx_wide_workspace_bytes(const MxWidePlan& p, int64_t M, int64_t N, int64_t K,
                                      bool qq) {
  const size_t pack = qq ? (mx_pack_bytes(M, K) + 255) & ~(size_t)255 : 0;
  return pack + (p.splits > 1 ? (size_t)p.splits * (size_t)M * (size_t)N * sizeof(float) : 0);
}

// Whether a product runs on the tile: above 16 rows, where the skinny kernel
// would read the weights again for every 16; with row identity above 32.
inline bool mx_wide_route(int64_t M, int64_t N, int64_t K, bool row_identity) {
  return M > (row_identity ? 32 : 16) && mx_wide_fits(M, N, K);
}

// Device workspace of mq_mxfp4_matmul / mq_mxfp4_qqmm.
inline size_t mx_workspace_bytes(int64_t M, int64_t N, int64_t K, bool qq, int cus,
                                 bool row_identity) {
  if (!mx_wide_route(M, N, K, row_identity)) return 0;
  return mx_wide_workspace_bytes(mx_wide_plan(M, N, K, qq, cus), M, N, K, qq);
}

// gather_qmm over P (x batch, expert) pairs on the skinny kernel; ws as
// gather_workspace_bytes(P, M) says.
template <int DT>
struct MxGatherLaunch {
  static int run(const void* x, const uint32_t* w, const uint8_t* s, const int32_t* lhs,
                 const int32_t* rhs, void* out, int64_t P, int64_t B, int64_t M, int64_t N,
                 int64_t K, int64_t E, void* ws, hipStream_t st, int* nlaunch);
};

// The same on the MFMA tile (mx_grouped.cuh), for calls that use a workspace;
// kStatusUnsupported beyond its address ranges.
template <int DT>
struct MxGroupedLaunch {
  static int run(const void* x, const uint32_t* w, const uint8_t* s, const int32_t* lhs,
                 const int32_t* rhs, void* out, int64_t P, int64_t B, int64_t M, int64_t N,
                 int64_t K, int64_t E, void* ws, hipStream_t st, int* nlaunch);
};

}  // namespace mq
