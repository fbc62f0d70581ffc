// Launchers of the dense gated feed-forward block (glu.cuh, glu_wide.cuh) and of
// products past quantized weights (qmm_grad.cuh), shared by their translation
// units and the C ABI.
#pragma once
#include "launch.h"

namespace mq {

enum GluAct { kActSilu = 0, kActGeluTanh = 1 };

// the tanh GELU: g / (1 + exp(-kGeluZ (g + kGeluCubic g^3))), kGeluZ = 2 sqrt(2 / pi)
constexpr float kGeluZ = 1.5957691216057308f, kGeluCubic = 0.044715f;

// out[M, N] = act(x . Wg^T) * (x . Wu^T); gf and uf (both or neither): the two
// products in float, [M, N].
struct GluArgs {
  const void* x;
  const uint32_t* wg;
  const void *sg, *bg;
  const uint32_t* wu;
  const void *su, *bu;
  void* out;
  float *gf, *uf;
  int64_t M, N, K;
  int act;
};

// Rows m0 .. m0 + M - 1 (M <= kGluSkinnyRows), one launch, with K in the slices that a
// launch of `rows` rows (M or more) needs: its sums' order.
constexpr int kGluSkinnyRows = 16;
template <int DT, int BITS, int GS>
struct GluSkinnyLaunch {
  static int run(const GluArgs& a, int64_t m0, int64_t M, int64_t rows, hipStream_t st);
};

// One row, in waves of 4 rows of either matrix (qmv_quad.cuh), one launch;
// kStatusUnsupported where a row's scales are too many for its LDS.
template <int DT, int BITS, int GS>
struct GluQuadLaunch {
  static int run(const GluArgs& a, hipStream_t st);
};

// All rows on the MFMA tile, 64 .. 256 rows by 128 columns of both matrices; with
// plan.splits > 1 over K splits, whose float planes ws holds.
template <int DT, int BITS, int GS>
struct GluWideLaunch {
  static int run(const GluArgs& a, const WidePlan& plan, void* ws, hipStream_t st, int* nlaunch);
};

inline bool glu_wide_eligible(int64_t M, int64_t K) {
  return K % 64 == 0 && K * 2 * 256 < ((int64_t)1 << 31) && M <= ((int64_t)65535) * 64;
}

// Floats of a row of a split's plane: whole eights, so that planes are written and summed
// four columns at a time whatever N is (N=9001, 45 rows: 5.2 us a sum before).
__host__ __device__ inline int64_t glu_plane(int64_t N) { return (N + 7) / 8 * 8; }

inline WidePlan glu_wide_plan(int64_t M, int64_t N, int64_t K, int bits, int cus, int max_splits) {
  return wide_plan(M, 2 * N, K, bits, cus, max_splits);
}

// Whether the MFMA tile runs.  row_identity (mq_set_row_identity): calls of up to 32 rows all
// run launches of the few-row kernel in the slices of its 16.
inline bool glu_wide_route(int64_t M, int64_t K, bool row_identity) {
  return M > (row_identity ? 32 : kGluSkinnyRows) && glu_wide_eligible(M, K);
}

inline size_t glu_workspace_bytes(int64_t M, int64_t N, int64_t K, int bits, int cus,
                                  bool row_identity) {
  if (!glu_wide_route(M, K, row_identity)) return 0;
  const WidePlan p = glu_wide_plan(M, N, K, bits, cus, 16);
  return p.splits > 1 ? (size_t)p.splits * 2 * (size_t)M * (size_t)glu_plane(N) * sizeof(float) : 0;
}

// ---- gradients past the weights ---------------------------------------------

// Steps of 64 weight rows that N rows take.
inline int64_t grad_steps(int64_t N) { return (N + 63) / 64; }

// dgu[M, 4 * P] (T), P = 64 * grad_steps(N): dg = d * u * act'(g), du = d * act(g), rounded
// to T, then what the rounding left of each, rounded to T; zeros past N columns
// (glu_grad.hip).  float16: rows times a power of two, undo[M] its reciprocal.
int launch_glu_grad(const void* d, const float* gf, const float* uf, void* dgu, float* undo,
                    int64_t M, int64_t N, int act, int dtype, hipStream_t st);

// Rows of N elements of a 16-bit type to rows of 64 * grad_steps(N), zeros past N.
int launch_pad_rows(const void* d, void* out, int64_t M, int64_t N, hipStream_t st);

// out[M, K] = d . W1, or with w2 dg . W1 + du . W2 of glu_grad.hip's rows, for quantized
// W [N, K]; d's rows of ld elements, padded to whole steps of 64 columns with zeros.  undo:
// glu_grad.hip's, with w2 and float16.
struct GradArgs {
  const void* d;
  int64_t ld;
  const uint32_t* w1;
  const void *s1, *b1;
  const uint32_t* w2;
  const void *s2, *b2;
  const float* undo;
  void* out;
  int64_t M, N, K;
};

template <int DT, int BITS, int GS>
struct GradLaunch {
  static int run(const GradArgs& a, const WidePlan& plan, void* ws, hipStream_t st, int* nlaunch);
};

// A tile's rows of out: with two matrices half its height, as each has two rows of d.
constexpr int grad_tile_rows(int bm, bool pair) { return pair ? bm / 2 : bm; }

// Elements of a row of d that the product reads: whole steps, of both matrices two numbers a
// column.
inline int64_t grad_row(int64_t N, int banks) { return (banks == 2 ? 4 : 1) * 64 * grad_steps(N); }

// One tile's rows of d (ld elements each), and the matrices in whole steps of rows, must fit
// 31-bit buffer ranges.
inline bool grad_eligible(int64_t M, int64_t N, int64_t K, int bits, int64_t ld, int banks = 1) {
  return 64 * grad_steps(N) * (K * bits / 8) < ((int64_t)1 << 31) &&
         ld * 2 * grad_tile_rows(256, banks == 2) < ((int64_t)1 << 31) &&
         M <= (int64_t)65535 * grad_tile_rows(64, banks == 2);
}

// Tile height and split of the sum, the pair of least cost by a model fitted to 6600
// calls (1 to 2048 rows, six matrices of either width, every height and up to 48
// splits; rms 7%): us per tile and step as in wide_plan, tp with many tiles per CU;
// a second 64-row tile on a CU adds t2 per step to the first's; splits cost their sum.
// The plan so chosen is 1.5% (4 bits) and 2.1% (8 bits) off the best one measured,
// 26% at most; wide_plan's constants were 8% off, 56% at most.  Two matrices, whose tiles have
// half the rows, go by the same costs: over 24 calls (16 to 2048 rows, four pairs of
// matrices) the plan is at the best of 52 others in the geometric mean, 11% off at most.
inline WidePlan grad_plan(int64_t M, int64_t N, int64_t K, int bits, int banks, int cus,
                          int max_splits) {
  static const WideTileUs us[2][4] = {
      {{4.53, 0.94, 0.84}, {5.43, 1.04, 1.20}, {5.86, 1.24, 1.51}, {5.92, 1.51, 1.91}},
      {{6.63, 1.10, 1.29}, {7.59, 1.20, 1.39}, {8.82, 1.34, 1.61}, {9.27, 1.53, 2.00}}};
  static const double t2[2] = {0.72, 1.13}, sum_us[2] = {5.97, 4.57}, mb_us[2] = {6.6, 7.7};
  const int w = bits == 8;
  const int64_t ns = banks * grad_steps(N), cols = (K + 255) / 256;
  WidePlan best;
  for (int sp = 1; sp <= max_splits; ++sp) {
    const double steps = (double)((ns + sp - 1) / sp);
    if (sp > 1 && steps < 4) break;
    for (int i = 3; i >= 0; --i) {
      const int bm = 64 * (i + 1), rows = grad_tile_rows(bm, banks == 2);
      const double tiles = (double)(cols * ((M + rows - 1) / rows) * sp);
      const double rounds = (double)(int64_t)((tiles + cus - 1) / cus);
      const WideTileUs& u = us[w][i];
      double cost = bm == 64 ? u.c0 * (double)((int64_t)(rounds + 1) / 2) +
                                   steps * (u.t + (rounds - 1) * t2[w])
                             : rounds * (u.c0 + u.t * steps);
      const double held = u.c0 + tiles / cus * u.tp * steps;
      if (held > cost) cost = held;
      if (sp > 1) cost += sum_us[w] + (8.0 * sp + 2.0) * (double)M * (double)K / (mb_us[w] * 1.0e6);
      if (best.cost_us == 0.0 || cost < best.cost_us) {
        best.bm = bm;
        best.splits = sp;
        best.cost_us = cost;
      }
    }
  }
  return best;
}

constexpr int kGradSplits = 48;

// Workspace of a product past one matrix (banks 1) or two: d's padded rows where N is
// not whole steps (banks 2: undo, then dgu), then the split planes.
inline size_t grad_undo_bytes(int64_t M, int banks) {
  return banks == 2 ? ((size_t)M * 4 + 255) & ~(size_t)255 : 0;
}
inline size_t grad_rows_bytes(int64_t M, int64_t N, int banks) {
  if (banks == 1 && N % 64 == 0) return 0;
  return grad_undo_bytes(M, banks) +
         (((size_t)M * (size_t)grad_row(N, banks) * 2 + 255) & ~(size_t)255);
}
inline size_t grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int bits, int banks, int cus) {
  return grad_rows_bytes(M, N, banks) +
         wide_workspace_bytes(grad_plan(M, N, K, bits, banks, cus, kGradSplits), M, K);
}

}  // namespace mq
