// W8A8 linear on the 5th-generation tensor core (tcgen05 kind::i8, sm_100a).
//
//   out[t][n] = (sum_k q[t][k] * w[n][k]) * s[t] * sw[n]
//
// q: int8 rows [T][K] with one fp32 scale each (kw8_add_rms_norm makes them);
// w: W8 weight [N][K].  Both operands are int8, so nothing is widened: TMA
// stages them and the tensor core reads both from shared memory.  Products and
// sums are exact in int32 (K <= kQ8MaxK); the result takes one rounding to
// fp32, two scale products and, for bf16, one more rounding.
#pragma once

#include "common.cuh"

namespace kw8 {

// |q|, |w| <= 128: 128 * 128 * K < 2^31.
constexpr int64_t kQ8MaxK = 131056;

struct Q8LinearArgs {
  int T, N, K;
  const float* x_scale;  // [T]
  const void* w_scale;   // 1 or [N]
  int w_scale_dtype, w_scale_pc;
  void* out;  // [T][N]
  int out_f32;
  // Pipeline, filled in by the launcher.
  int nt;          // columns of a tile (multiple of 16)
  int stages;      // ring depth
  int k_splits;    // CTAs of a cluster that share one tile's k range
  int w_tiled;     // weights in the tiled layout
};

int launch_linear_q8(const int8_t* q, const kw8_weight& w, const Q8LinearArgs& args, cudaStream_t stream);

}  // namespace kw8
