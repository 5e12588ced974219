// Token sampling from logits (see sample.cu).
#pragma once

#include "common.cuh"

namespace kw8 {

constexpr int64_t kSampleMaxV = 8 * 49152;  // sixteen CTAs' shared memory holds it in fp32, eight nearly (387360)

struct SampleArgs {
  const void* logits;  // row r at logits + r * ld
  int64_t ld;
  int V;
  const float* u;
  const float *temperature, *top_p, *min_p;  // one per row, or null: the values below
  const int32_t* top_k;
  float temperature0, top_p0, min_p0;
  int32_t top_k0;
  int32_t* token;
  float* logprob;  // or null
  int slice;       // logits per CTA, filled in by the launcher
};

int launch_sample(const SampleArgs& args, int64_t B, int logits_dtype, cudaStream_t stream);

}  // namespace kw8
