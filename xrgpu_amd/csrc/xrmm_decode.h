// Rotary positions and the draw of tokens: argument blocks of their launches.
#pragma once
#include "xrmm_lowbit.h"

namespace xrmm {

// q and k [rows, heads, D] (k may have no heads), turned into oq and ok; token strides in elements.
struct RopeArgs {
  const void *q, *k;
  void *oq, *ok;
  int64_t q_stride, k_stride, oq_stride, ok_stride;
  const double* freq;        // [R / 2], radians a position
  const void* positions;     // [rows] int32 or int64, or null: the last rows of sequences as the cache's calls have them
  const int32_t* lengths;    // [B]
  const int32_t* starts;     // [B + 1], or null: `each` rows a sequence
  double magnitude;
  int64_t rows, row0;        // row0: the first of a launch
  int32_t B, each, Hq, Hk, D, R;
  int dtype;                 // LT
  bool wide_positions, interleaved, inverse;
};

// A token for each row of logits [rows, V].
struct SampleArgs {
  const void* x;
  const float* u;
  // a value for each row, or null: the one for all
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  double temperature1, top_p1, min_p1;
  int32_t top_k1;
  int32_t* tokens;
  float* shares;             // logarithms of the drawn tokens' shares
  void* ws;
  int64_t ws_bytes, stride, rows;
  int32_t V;
  int dtype;                 // LT
};

// Threads of a launch of a call that takes several (see grid_counts).
constexpr int64_t kLaunchThreads = int64_t{1} << 31;

hipError_t launch_rope(const RopeArgs& a, hipStream_t st);
hipError_t launch_sample(const SampleArgs& a, hipStream_t st);
int64_t sample_workspace_bytes(int64_t rows, int64_t V);

}  // namespace xrmm
