// RMSNorm (kappa/gemma3/norms.py:8-13 with Gemma's (1 + scale),
// kappa/qwen3/norms.py:10-16 with Qwen's scale) and the residual epilogue of
// the FFN sub-block (kappa/gemma3/block.py:73-82, kappa/qwen3/block.py:68-81).
//
// A CTA takes up to 256 / tpr rows, tpr threads per row (the fewest, from
// 32, that hold the row in at most kNormMaxVec 8-wide vectors each: one
// warp per 2048-wide row), fewer rows when the grid would otherwise have
// under two CTAs per SM.  The row is read once into registers,
// the sum of squares is reduced over the row's threads in fp32 (a fixed
// order), and the row is written once.  Rounding follows kappa: the norm computes in fp32 and rounds its
// output to the activation dtype once; the FFN output is rounded to bf16
// before the post-FFN norm, and the residual add rounds once more.
#include "norm.cuh"

namespace kw8 {

namespace {

// Sum of v over the tpr threads of this thread's row group (every thread
// of the CTA calls it; the result is the same in every thread of a group).
__device__ __forceinline__ float group_sum(float v, float* red, int tpr) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // red may still be read by an earlier call
  if (lane == 0) red[warp] = v;
  __syncthreads();
  const int wpg = tpr >> 5, first = (warp / wpg) * wpg;
  float s = 0.f;
  for (int w = 0; w < wpg; ++w) s += red[first + w];  // the same order in every thread
  return s;
}

__device__ __forceinline__ void bf16x8_to_f32(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

__device__ __forceinline__ uint4 f32x8_to_bf16(const float (&f)[8]) {
  uint4 o;
  uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    ow[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return o;
}

// g[d] of the norm: 1 + scale (Gemma) or scale (Qwen), in fp32.
__device__ __forceinline__ float norm_gain(const void* scale, int dtype, int kind, int64_t d) {
  const float s = load_scale(scale, dtype, d);
  return kind == KW8_NORM_GEMMA ? 1.0f + s : s;
}

// v (this thread's nv vectors of the row, fp32) <- (v * r) * g, r from the
// row's mean square.
__device__ __forceinline__ void rms_apply(float (&v)[kNormMaxVec][8], int nv, int64_t D,
                                          const void* scale, int dtype, int kind, float eps,
                                          float* red, int tpr, int tl) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < kNormMaxVec; ++j)
    if (j < nv)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[j][i], v[j][i], ss);
  const float total = group_sum(ss, red, tpr);
  const float r = rsqrtf(__fdiv_rn(total, static_cast<float>(D)) + eps);
#pragma unroll
  for (int j = 0; j < kNormMaxVec; ++j) {
    if (j >= nv) continue;
    const int64_t d0 = (static_cast<int64_t>(j) * tpr + tl) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = __fmul_rn(__fmul_rn(v[j][i], r), norm_gain(scale, dtype, kind, d0 + i));
  }
}

__global__ void __launch_bounds__(kNormThreads)
    rms_norm_kernel(const uint4* __restrict__ x, int64_t T, int64_t D, const void* __restrict__ scale, int dtype,
                    int kind, float eps, int tpr, uint4* __restrict__ out) {
  __shared__ float red[kNormThreads / 32];
  const int64_t vec = D / 8;
  const int tl = threadIdx.x % tpr;
  const int64_t row = blockIdx.x * static_cast<int64_t>(blockDim.x / tpr) + threadIdx.x / tpr;
  const int nv = row < T ? static_cast<int>((vec - tl + tpr - 1) / tpr) : 0;
  const uint4* xr = x + row * vec;
  float v[kNormMaxVec][8];
#pragma unroll
  for (int j = 0; j < kNormMaxVec; ++j)
    if (j < nv) bf16x8_to_f32(xr[j * tpr + tl], v[j]);
  rms_apply(v, nv, D, scale, dtype, kind, eps, red, tpr, tl);
  uint4* orow = out + row * vec;
#pragma unroll
  for (int j = 0; j < kNormMaxVec; ++j)
    if (j < nv) orow[j * tpr + tl] = f32x8_to_bf16(v[j]);
}

__global__ void __launch_bounds__(kNormThreads)
    block_finish_kernel(const float4* __restrict__ part, int splits, int64_t stride4, int64_t T, int64_t D,
                        const void* __restrict__ scale, int dtype, int kind, float eps,
                        const uint4* __restrict__ h, int tpr, uint4* __restrict__ out) {
  __shared__ float red[kNormThreads / 32];
  const int64_t vec = D / 8;
  const int tl = threadIdx.x % tpr;
  const int64_t row = blockIdx.x * static_cast<int64_t>(blockDim.x / tpr) + threadIdx.x / tpr;
  const int nv = row < T ? static_cast<int>((vec - tl + tpr - 1) / tpr) : 0;
  float v[kNormMaxVec][8];
#pragma unroll
  for (int j = 0; j < kNormMaxVec; ++j) {
    if (j >= nv) continue;
    const int64_t e4 = (row * vec + j * tpr + tl) * 2;  // float4 index
    float4 a = part[e4], b = part[e4 + 1];
    for (int s = 1; s < splits; ++s) {
      const float4 c = part[s * stride4 + e4], d = part[s * stride4 + e4 + 1];
      a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
      b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
    }
    const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = __bfloat162float(__float2bfloat16_rn(f[i]));  // the FFN output in bf16
  }
  if (scale != nullptr) {
    rms_apply(v, nv, D, scale, dtype, kind, eps, red, tpr, tl);
#pragma unroll
    for (int j = 0; j < kNormMaxVec; ++j)
      if (j < nv)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = __bfloat162float(__float2bfloat16_rn(v[j][i]));
  }
#pragma unroll
  for (int j = 0; j < kNormMaxVec; ++j) {
    if (j >= nv) continue;
    const int64_t e = row * vec + j * tpr + tl;
    if (h != nullptr) {
      float hv[8];
      bf16x8_to_f32(h[e], hv);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = __fadd_rn(hv[i], v[j][i]);
    }
    out[e] = f32x8_to_bf16(v[j]);
  }
}

// Largest bit pattern over the tpr threads of this thread's row group.
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* red, int tpr) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (tpr == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) red[warp] = v;  // not the array of group_sum: no barrier needed before
  __syncthreads();
  const int wpg = tpr >> 5, first = (warp / wpg) * wpg;
  for (int w = 0; w < wpg; ++w) v = max(v, red[first + w]);
  return v;
}

// The larger of a and |b|; NaN if either is.
__device__ __forceinline__ float max_abs_nan(float a, float b) {
  float d;
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Residual add + RMSNorm + optional 8-bit rows (definition in norm.cuh).
// One pass, a CTA per row: the row stays in its threads' registers (kVec 8-wide vectors per
// thread at most) between the sum of squares, the absmax and the stores, so
// each input is read once and each output written once.  HBM is the bound, with
// the issue slots close behind (about 13 instructions per value), hence the
// shifts for divisions and 32-bit indexes inside a row.
// The absmax keeps NaN (max.NaN), and its bit pattern is ordered like the value
// with infinity and NaN above every number, so one integer reduction also finds
// the rows that are not finite.  Rounding to int8 is one fma: y * (1/s) + 1.5 *
// 2^23 leaves the nearest integer (ties to even), in two's complement, in the
// low byte of the sum's bits.  1/s rounds once, so a value within about 2^-16 of
// a half step may round to the other side of it than an exact division would.
template <int kVec, bool kAdd, bool kQ8, bool kF32Gain>
__global__ void __launch_bounds__(kNormThreads)
    add_rms_norm_kernel(const uint4* x, const uint4* residual, int vec, const uint4* __restrict__ scale,
                        float bias, float eps, int tpr_log2, uint4* h_out, uint4* y_out, uint2* q_out, float* s_out) {
  __shared__ float red[kNormThreads / 32];
  __shared__ uint32_t red_max[kNormThreads / 32];
  const int tpr = 1 << tpr_log2, tl = static_cast<int>(threadIdx.x);
  const int64_t row = blockIdx.x;
  const int nv = (vec - tl + tpr - 1) >> tpr_log2;
  const int64_t e0 = row * vec + tl;
  uint4 a[kVec], b[kAdd ? kVec : 1];
#pragma unroll
  for (int j = 0; j < kVec; ++j)
    if (j < nv) {
      a[j] = (x + e0)[j << tpr_log2];
      if constexpr (kAdd) b[j] = (residual + e0)[j << tpr_log2];
    }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < kVec; ++j)
    if (j < nv) {
      float f[8];
      bf16x8_to_f32(a[j], f);
      if constexpr (kAdd) {
        float r[8];
        bf16x8_to_f32(b[j], r);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += r[i];
        a[j] = f32x8_to_bf16(f);  // the residual stream is kept in bf16, and normed as it is kept
        if (h_out != nullptr) (h_out + e0)[j << tpr_log2] = a[j];
        bf16x8_to_f32(a[j], f);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
    }
  const float total = group_sum(ss, red, tpr);
  const float r = rsqrtf(__fdiv_rn(total, static_cast<float>(vec * 8)) + eps);
  float v[kVec][8];
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < kVec; ++j)
    if (j < nv) {
      if constexpr (!kAdd)
        if (h_out != nullptr) (h_out + e0)[j << tpr_log2] = a[j];
      float g[8];
      if constexpr (kF32Gain) {
        const uint4* p = scale + 2 * ((j << tpr_log2) + tl);
        const uint4 lo = __ldg(p), hi = __ldg(p + 1);
        const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = __uint_as_float(w[i]);
      } else {
        bf16x8_to_f32(__ldg(scale + (j << tpr_log2) + tl), g);
      }
      bf16x8_to_f32(a[j], v[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = __fmul_rn(__fmul_rn(v[j][i], r), g[i] + bias);  // g = scale + 1 (Gemma) or + 0
        if constexpr (kQ8) top = max_abs_nan(top, v[j][i]);
      }
      if constexpr (!kQ8) (y_out + e0)[j << tpr_log2] = f32x8_to_bf16(v[j]);
    }
  if constexpr (kQ8) {
    const uint32_t bits = group_max(__float_as_uint(top), red_max, tpr);
    const bool finite = bits < 0x7F800000u;
    const float s = finite ? fmaxf(__fdiv_rn(__uint_as_float(bits), 127.0f), 1.17549435e-38f)
                           : __uint_as_float(0x7FC00000u);
    const float inv = __fdiv_rn(1.0f, s);
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (j < nv) {
        uint32_t m[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = __float_as_uint(fmaf(v[j][i], inv, 12582912.0f));
        uint2 o;
        o.x = __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410);
        o.y = __byte_perm(__byte_perm(m[4], m[5], 0x0040), __byte_perm(m[6], m[7], 0x0040), 0x5410);
        (q_out + e0)[j << tpr_log2] = finite ? o : make_uint2(0u, 0u);
      }
    if (tl == 0) s_out[row] = s;
  }
}

// Threads per row: the fewest of 32, 64, 128, 256 that hold a row in at most
// kNormMaxVec vectors each, doubled while the rows would keep fewer than
// ~131k threads busy (few rows: more threads per row; measured at T = 256 /
// 4096, D = 2560 / 2048).
int norm_tpr(int64_t T, int64_t D) {
  const int64_t vec = D / 8;
  int tpr = 32;
  while (tpr < kNormThreads && (vec + tpr - 1) / tpr > kNormMaxVec) tpr *= 2;
  while (tpr < kNormThreads && tpr < vec && T * tpr < 148 * 896) tpr *= 2;
  return tpr;
}

// Rows per CTA: as many as kNormThreads threads hold, fewer when that would
// leave fewer than two CTAs per SM (few rows: T = 256 gets one row a CTA).
int64_t norm_rows_per_cta(int64_t T, int tpr) {
  int64_t rpc = kNormThreads / tpr;
  while (rpc > 1 && (T + rpc - 1) / rpc < 2 * 148) rpc /= 2;
  return rpc;
}

int check_norm(int64_t T, int64_t D, int scale_dtype, int kind, float eps) {
  KW8_REQUIRE(T >= 0 && D >= 8 && D % 8 == 0 && D <= kNormMaxD, KW8_ERR_UNSUPPORTED,
              "RMSNorm rows need D %% 8 == 0 and 8 <= D <= %lld (D=%lld)", (long long)kNormMaxD,
              (long long)D);
  KW8_REQUIRE(T < (1ll << 31), KW8_ERR_UNSUPPORTED, "too many rows");
  KW8_REQUIRE(scale_dtype == KW8_DT_F32 || scale_dtype == KW8_DT_BF16, KW8_ERR_INVALID_ARG,
              "norm scale dtype must be f32 or bf16");
  KW8_REQUIRE(kind == KW8_NORM_GEMMA || kind == KW8_NORM_QWEN, KW8_ERR_INVALID_ARG, "unknown norm kind %d",
              kind);
  KW8_REQUIRE(eps >= 0.f, KW8_ERR_INVALID_ARG, "eps must be >= 0");
  return KW8_OK;
}

}  // namespace

int launch_rms_norm(const void* x, int64_t T, int64_t D, const void* scale, int scale_dtype, int kind,
                    float eps, void* out, cudaStream_t stream) {
  KW8_REQUIRE(x && scale && out, KW8_ERR_INVALID_ARG, "null pointer");
  int rc = check_norm(T, D, scale_dtype, kind, eps);
  if (rc) return rc;
  KW8_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
              KW8_ERR_UNSUPPORTED, "RMSNorm rows must be 16-byte aligned");
  if (T == 0) return KW8_OK;
  const int tpr = norm_tpr(T, D);
  const int64_t rpc = norm_rows_per_cta(T, tpr);
  rms_norm_kernel<<<static_cast<unsigned>((T + rpc - 1) / rpc), static_cast<unsigned>(rpc * tpr), 0, stream>>>(
      static_cast<const uint4*>(x), T, D, scale, scale_dtype, kind, eps, tpr, static_cast<uint4*>(out));
  KW8_CHECK_LAUNCH();
  return KW8_OK;
}

int launch_block_finish(const float* part, int splits, int64_t split_stride, int64_t T, int64_t D,
                        const void* post_scale, int scale_dtype, int kind, float eps, const void* h,
                        void* out, cudaStream_t stream) {
  KW8_REQUIRE(part && out && splits >= 1, KW8_ERR_INVALID_ARG, "null pointer");
  int rc = check_norm(T, D, scale_dtype, kind, eps);
  if (rc) return rc;
  KW8_REQUIRE(split_stride % 4 == 0 &&
                  ((reinterpret_cast<uintptr_t>(part) | reinterpret_cast<uintptr_t>(out) |
                    reinterpret_cast<uintptr_t>(h)) & 15) == 0,
              KW8_ERR_UNSUPPORTED, "block epilogue rows must be 16-byte aligned");
  if (T == 0) return KW8_OK;
  const int tpr = norm_tpr(T, D);
  const int64_t rpc = norm_rows_per_cta(T, tpr);
  block_finish_kernel<<<static_cast<unsigned>((T + rpc - 1) / rpc), static_cast<unsigned>(rpc * tpr), 0, stream>>>(
      reinterpret_cast<const float4*>(part), splits, split_stride / 4, T, D, post_scale, scale_dtype, kind, eps,
      static_cast<const uint4*>(h), tpr, static_cast<uint4*>(out));
  KW8_CHECK_LAUNCH();
  return KW8_OK;
}

namespace {

struct AddNormArgs {
  const void *x, *residual, *scale;
  int T, vec;
  bool f32_gain;
  float bias, eps;
  int tpr_log2;
  void *h_out, *y_out;
  int8_t* q_out;
  float* s_out;
};

template <int kVec, bool kAdd, bool kQ8>
int launch_add_rms_norm_vec(const AddNormArgs& a, cudaStream_t stream) {
  auto kernel = a.f32_gain ? add_rms_norm_kernel<kVec, kAdd, kQ8, true> : add_rms_norm_kernel<kVec, kAdd, kQ8, false>;
  kernel<<<static_cast<unsigned>(a.T), 1u << a.tpr_log2, 0, stream>>>(static_cast<const uint4*>(a.x), static_cast<const uint4*>(a.residual), a.vec,
                                     static_cast<const uint4*>(a.scale), a.bias, a.eps, a.tpr_log2,
                                     static_cast<uint4*>(a.h_out), static_cast<uint4*>(a.y_out),
                                     reinterpret_cast<uint2*>(a.q_out), a.s_out);
  KW8_CHECK_LAUNCH();
  return KW8_OK;
}

template <int kVec>
int launch_add_rms_norm_any(const AddNormArgs& a, cudaStream_t stream) {
  if (a.residual) return a.q_out ? launch_add_rms_norm_vec<kVec, true, true>(a, stream)
                                 : launch_add_rms_norm_vec<kVec, true, false>(a, stream);
  return a.q_out ? launch_add_rms_norm_vec<kVec, false, true>(a, stream)
                 : launch_add_rms_norm_vec<kVec, false, false>(a, stream);
}

}  // namespace

int launch_add_rms_norm(const void* x, const void* residual, int64_t T, int64_t D, const void* scale,
                        int scale_dtype, int kind, float eps, void* h_out, void* y_out, int8_t* q_out,
                        float* s_out, cudaStream_t stream) {
  int rc = check_norm(T, D, scale_dtype, kind, eps);
  if (rc || T == 0) return rc;
  KW8_REQUIRE(x && scale, KW8_ERR_INVALID_ARG, "null x/scale");
  KW8_REQUIRE((y_out != nullptr) != (q_out != nullptr) && (q_out != nullptr) == (s_out != nullptr),
              KW8_ERR_INVALID_ARG, "the norm writes either bf16 rows or int8 rows with their scales");
  KW8_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                reinterpret_cast<uintptr_t>(h_out) | reinterpret_cast<uintptr_t>(y_out)) & 15) == 0 &&
                  (reinterpret_cast<uintptr_t>(q_out) & 7) == 0 && (reinterpret_cast<uintptr_t>(s_out) & 3) == 0,
              KW8_ERR_UNSUPPORTED, "RMSNorm rows must be 16-byte aligned (int8 rows 8-byte)");
  KW8_REQUIRE((reinterpret_cast<uintptr_t>(scale) & 15) == 0, KW8_ERR_UNSUPPORTED,
              "the norm's scale must be 16-byte aligned");
  // Outputs: h over its own input element by element, or no overlap at all.
  const int64_t n2 = T * D * 2, out_bytes = q_out ? T * D : n2;
  const void* out = q_out ? static_cast<const void*>(q_out) : y_out;
  bool bad = overlaps(out, out_bytes, x, n2) || overlaps(out, out_bytes, residual, n2) ||
             overlaps(out, out_bytes, h_out, n2) || overlaps(s_out, T * 4, out, out_bytes) ||
             overlaps(s_out, T * 4, h_out, n2) || overlaps(s_out, T * 4, x, n2) || overlaps(s_out, T * 4, residual, n2);
  for (const void* in : {x, residual}) bad = bad || (h_out != in && overlaps(h_out, n2, in, n2));
  const int64_t scale_bytes = D * (scale_dtype == KW8_DT_F32 ? 4 : 2);
  bad = bad || overlaps(scale, scale_bytes, out, out_bytes) || overlaps(scale, scale_bytes, h_out, n2) ||
        overlaps(scale, scale_bytes, s_out, T * 4);
  KW8_REQUIRE(!bad, KW8_ERR_INVALID_ARG, "the norm's outputs overlap its inputs or one another");
  AddNormArgs a{};
  a.x = x;
  a.residual = residual;
  a.scale = scale;
  a.T = static_cast<int>(T);
  a.vec = static_cast<int>(D / 8);
  a.f32_gain = scale_dtype == KW8_DT_F32;
  a.bias = kind == KW8_NORM_GEMMA ? 1.f : 0.f;
  a.eps = eps;
  a.h_out = h_out;
  a.y_out = y_out;
  a.q_out = q_out;
  a.s_out = s_out;
  // Threads per row: the fewest that hold it in five vectors each, more while
  // the rows would keep few threads busy.  A row per CTA, so that no row waits
  // for another's reductions (8192 x 2560 with residual to int8 rows: one row
  // per CTA 27.1 us, four 27.8; without residual 17.5 against 19.5; 4096 x 2048:
  // 12.3 against 13.2).
  int tpr = 32;
  while (tpr < kNormThreads && (a.vec + tpr - 1) / tpr > 5) tpr *= 2;
  while (tpr < kNormThreads && tpr < a.vec && T * tpr < 148 * 896) tpr *= 2;
  while ((1 << a.tpr_log2) < tpr) ++a.tpr_log2;
  const int per = (a.vec + tpr - 1) / tpr;  // 8-wide vectors per thread
  if (per <= 1) return launch_add_rms_norm_any<1>(a, stream);
  if (per <= 2) return launch_add_rms_norm_any<2>(a, stream);
  if (per <= 3) return launch_add_rms_norm_any<3>(a, stream);
  if (per <= 5) return launch_add_rms_norm_any<5>(a, stream);
  return launch_add_rms_norm_any<kNormMaxVec>(a, stream);
}

}  // namespace kw8
