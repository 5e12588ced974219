// RMSNorm and the residual epilogue of a decoder block's FFN (see norm.cu).
#pragma once

#include "common.cuh"

namespace kw8 {

// Rows of D (a multiple of 8, at most kNormMaxD) spread over CTAs of
// kNormThreads threads, each thread holding at most kNormMaxVec 8-wide vectors.
constexpr int kNormThreads = 256;
constexpr int kNormMaxVec = 8;  // 8-wide vectors per thread
constexpr int64_t kNormMaxD = static_cast<int64_t>(kNormThreads) * 8 * kNormMaxVec;

// out = bf16((f32(x) * rsqrt(mean(f32(x)^2) + eps)) * g), g = 1 + scale
// (kind KW8_NORM_GEMMA) or scale (KW8_NORM_QWEN); x, out bf16 [T][D].
int launch_rms_norm(const void* x, int64_t T, int64_t D, const void* scale, int scale_dtype,
                    int kind, float eps, void* out, cudaStream_t stream);

// The end of the FFN sub-block, row by row:
//   y   = bf16(sum over s < splits of part[s][t])   (the FFN output, fp32 partials)
//   y   = rms_norm(y, post_scale)                   (if post_scale != nullptr)
//   out = bf16(f32(h[t]) + f32(y))                  (if h != nullptr; else out = y)
int launch_block_finish(const float* part, int splits, int64_t split_stride, int64_t T, int64_t D,
                        const void* post_scale, int scale_dtype, int kind, float eps,
                        const void* h, void* out, cudaStream_t stream);

// The norm with the residual's addition in front and, optionally, 8-bit rows
// behind it.  Per row of D values:
//   h = residual ? bf16(f32(x) + f32(residual)) : x     (stored to h_out if given)
//   y = (f32(h) * rsqrt(mean(f32(h)^2) + eps)) * g      (fp32)
//   q_out == nullptr:  y_out = bf16(y)
//   else:  s = max(max|y| / 127, FLT_MIN),  q_out = round_half_even(y * (1 / s)),  s_out[row] = s.
// A row whose y is not finite gets q = 0 and s = NaN.  h_out may be x or
// residual (in place); otherwise the outputs overlap nothing.
int launch_add_rms_norm(const void* x, const void* residual, int64_t T, int64_t D, const void* scale,
                        int scale_dtype, int kind, float eps, void* h_out, void* y_out, int8_t* q_out,
                        float* s_out, cudaStream_t stream);

}  // namespace kw8
