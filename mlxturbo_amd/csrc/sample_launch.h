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
  int tile;                                     // log2 of a tile's 16-byte granules
  int32_t* token;
  float* logprob;
};

// Rows of one sequence of launches, whose workspace they share.
constexpr int kSampleRows = 256;

// Chunks of a row: about 1024 workgroups over the rows of a sequence, of 4096 words
// at least.
inline int sample_chunks(int64_t R, int64_t V) {
  const int64_t rows = R < kSampleRows ? R : kSampleRows;
  int64_t c = 1024 / (rows > 0 ? rows : 1);
  if (c > (V + 4095) / 4096) c = (V + 4095) / 4096;
  return c < 1 ? 1 : (int)c;
}

// A row's tiles: of 64 granules, or more where that would be over 1024 of them.
constexpr int kSampleTiles = 1024;
inline int sample_tile(int64_t V, int dtype) {
  const int64_t e = dtype == kF32 ? 4 : 8, n = (V + 2 * e - 2) / e;
  int tile = 6;
  while ((n + ((int64_t)1 << tile) - 1) >> tile > kSampleTiles) ++tile;
  return tile;
}

// A row's workspace: the tiles' first words and masses, masses of the bins, the list,
// the row's first word and bound, and counts of the bins, the list's length and the workgroups that are done.
constexpr int kSampleBins = 2048, kSampleList = 4096;
constexpr size_t kSampleRowBytes =
    (2 * kSampleTiles + kSampleBins + kSampleList + 2) * 8 + (kSampleBins + 4) * 4;

inline size_t sample_workspace_bytes(int64_t R) {
  return (size_t)(R < kSampleRows ? R : kSampleRows) * kSampleRowBytes;
}

int launch_sample(const SampleArgs& a, int dtype, void* ws, hipStream_t st, int* nlaunch);

}  // namespace mq
