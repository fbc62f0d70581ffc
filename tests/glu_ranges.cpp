// For each input line "bits gs N K": how the gated few-row kernel (glu.cuh) reads an [N, K]
// matrix's codes and scales, as "past read lds": the most bytes that a load reaches past them,
// whether every byte is read, and the most LDS that a launch of 1 to 16 rows takes.
#include <algorithm>
#include <cstdio>
#include <vector>

#include "glu.cuh"

namespace {

template <int BITS, int GS>
void report(int64_t N, int64_t K) {
  constexpr int UC = mq::GluGeom<BITS>::UC;
  const uint32_t rowB = (uint32_t)(K * BITS / 8);
  const int S = (int)((K + UC - 1) / UC), G = (int)(K / GS);
  int64_t past = 0;
  std::vector<char> code(N * rowB, 0), scale(N * G, 0);
  for (int64_t n0 = 0; n0 < N; n0 += mq::kGluCols) {
    for (int s = 0; s < S; ++s)
      for (int lane = 0; lane < 64; ++lane) {
        const int64_t at = (n0 + mq::glu_lane_row(lane, n0, (int)N)) * rowB + mq::glu_lane_byte(lane, s, rowB);
        past = std::max(past, at + 16 - N * (int64_t)rowB);
        for (int b = 0; b < 16; ++b)
          if (at + b < N * (int64_t)rowB) code[at + b] = 1;
      }
    // pieces of eights where whole rows are, and single ones
    for (int P : {G % 8 ? 1 : 8, 1})
      for (int64_t n = n0; n < n0 + mq::kGluCols; ++n)
        for (int g = 0; g < S * (UC / GS); g += P) {
          const int64_t at = std::min(n, N - 1) * G + mq::glu_piece_at(g, G, P);
          past = std::max(past, 2 * (at + P - N * G));
          for (int b = 0; b < P; ++b)
            if (at + b < N * G) scale[at + b] |= P == 1 ? 1 : 2;
        }
  }
  bool all = std::all_of(code.begin(), code.end(), [](char c) { return c != 0; });
  for (char c : scale) all &= (c & 1) && (G % 8 || (c & 2));
  // the launch's slices of x and scales (256 CUs)
  size_t lds = 0;
  const int64_t tiles = (N + mq::kGluCols - 1) / mq::kGluCols;
  for (int64_t M = 1; M <= mq::kGluSkinnyRows; ++M) {
    const mq::GluSlices p = mq::glu_slices<BITS, GS>(M, tiles, S, 256);
    lds = std::max(lds, p.lds);
  }
  printf("%lld %d %lld\n", (long long)past, (int)all, (long long)lds);
}

}  // namespace

int main() {
  long long bits, gs, N, K;
  while (scanf("%lld %lld %lld %lld", &bits, &gs, &N, &K) == 4) {
#define MQ_CASE(B, G) \
  if (bits == B && gs == G) report<B, G>(N, K);
    MQ_CASE(4, 32) MQ_CASE(4, 64) MQ_CASE(4, 128) MQ_CASE(8, 32) MQ_CASE(8, 64) MQ_CASE(8, 128)
#undef MQ_CASE
  }
  return 0;
}
