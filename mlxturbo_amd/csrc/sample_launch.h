// Launcher of the sampling kernels (sample.hip), shared with the C ABI.
#pragma once
#include <type_traits>

#include "launch.h"

namespace mq {

// R rows of V logits, row_stride elements apart; u [R].  A setting is an array of R
// values, or NULL and the one value for all rows.
struct SampleArgs {
  const void* logits;
  int64_t row_stride, R, V;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p;
  float temperature0, top_p0, min_p0;
  int32_t top_k0;
  double scale;                                 // mass of the most probable word
  int32_t* token;
  float* logprob;
};

// Rows of one sequence of launches, whose workspace they share.
constexpr int kSampleRows = 256;

// Chunks of a row: about 1024 workgroups over the rows of a sequence, of 2048 words
// at least.
inline int sample_chunks(int64_t R, int64_t V) {
  const int64_t rows = R < kSampleRows ? R : kSampleRows;
  int64_t c = 1024 / (rows > 0 ? rows : 1);
  if (c > (V + 2047) / 2048) c = (V + 2047) / 2048;
  return c < 1 ? 1 : (int)c;
}

// Bytes of a row's workspace: two arrays of C, masses of 2048 bins, a list of 4096, and
// 2048 counts and the list's length.
__host__ __device__ inline size_t sample_row_bytes(int C) {
  return ((size_t)C * 16 + 2048 * 8 + 4096 * 8 + 2049 * 4 + 15) & ~(size_t)15;
}

inline size_t sample_workspace_bytes(int64_t R, int64_t V) {
  return (size_t)(R < kSampleRows ? R : kSampleRows) * sample_row_bytes(sample_chunks(R, V));
}

int launch_sample(const SampleArgs& a, int dtype, void* ws, hipStream_t st, int* nlaunch);

}  // namespace mq
