// Launcher of the token sampler (returns 0 or a negative blt_status).
#pragma once
#include "rowops.hpp"

namespace blt {

// A setting of all rows, or (where the pointer is not null) of each.
struct SampleSetting {
  double temperature, top_p, min_p;
  int top_k;
  const float *temperatures, *top_ps, *min_ps;
  const int32_t* top_ks;
};
struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int dtype;
  int64_t rows;
  int vocab;
  const float* uniform;
  SampleSetting set;
  int32_t* out;
};
constexpr int kSampleVocab = 1 << 20;
int64_t sample_workspace_bytes(int64_t rows, int vocab);
int launch_sample(const SampleArgs& a, void* ws, hipStream_t s);

}  // namespace blt
