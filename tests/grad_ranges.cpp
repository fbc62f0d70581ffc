// For each input line "bits gs N K": how the gradient tile (qmm_grad.cuh) reads a [N, K]
// matrix, as "taken past beyond read" where
//   taken: the kernels take the size (0: the other numbers are 0);
//   past: the most bytes that a load in range reaches past the codes or scales;
//   beyond: the most bytes that a scalar offset is past the buffer's size, where the range
//     check (lane offset < size - scalar offset, in 32 bits) would wrap;
//   read: every row's first and last codes and scales are read.
#include <algorithm>
#include <cstdio>
#include <vector>

#include "qmm_grad.cuh"

namespace {

int64_t past, beyond;

// One load; whether it is in range.
bool load(uint32_t lane, uint32_t scalar, int size, int64_t bytes) {
  beyond = std::max(beyond, (int64_t)scalar - bytes);
  if (lane >= (uint32_t)bytes - scalar) return false;
  past = std::max(past, (int64_t)lane + scalar + size - bytes);
  return true;
}

template <int BITS, int GS>
void report(int64_t N, int64_t K) {
  past = beyond = 0;
  const bool taken = mq::grad_eligible(64, N, K, BITS, 64 * mq::grad_steps(N));
  std::vector<int> seen(taken ? N : 0, 0);
  const uint32_t rowB = (uint32_t)K * BITS / 8, rowS = (uint32_t)(K / GS) * 2;
  const int64_t wbytes = N * rowB, sbytes = N * rowS;
  // steps: the first two, and the last three
  const int64_t ns = taken ? mq::grad_steps(N) : 0;
  for (int64_t k = 0; k < ns; ++k) {
    if (k == 2) k = std::max<int64_t>(k, ns - 3);
    for (int col : {0, (int)K - 8}) {
      for (int s = 0; s < 4; ++s) {
        const uint32_t so = mq::grad_rows_at((uint32_t)(64 * k + 8 * s), rowB, wbytes);
        for (int lane = 0; lane < 8; ++lane)
          for (int e = 0; e < 2; ++e) {
            const uint32_t row = mq::grad_lane_row(lane) + e;
            if (load(row * rowB + (uint32_t)col * BITS / 8, so, BITS, wbytes)) {
              const int64_t n = ((int64_t)so + row * rowB) / rowB;
              if (n < N) seen[n] |= col ? 2 : 1;
            }
          }
      }
      const uint32_t so = mq::grad_rows_at((uint32_t)(64 * k), rowS, sbytes);
      for (uint32_t lane = 0; lane < 64; ++lane)
        if (load(lane * rowS + (uint32_t)(col / GS) * 2, so, 2, sbytes)) {
          const int64_t n = ((int64_t)so + lane * rowS) / rowS;
          if (n < N) seen[n] |= col ? 8 : 4;
        }
    }
  }
  bool all = true;
  for (int64_t n = 0; n < (int64_t)seen.size(); ++n)
    if (n < 128 || n >= 64 * (ns - 3)) all &= seen[n] == 15;
  printf("%d %lld %lld %d\n", (int)taken, (long long)past, (long long)beyond, (int)all);
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
