// Token sampling: temperature, top-k, top-p and min-p, from given random numbers.
//
// Per row of logits x (NaN counts as -inf), with m the largest:
//   w_i = floor(2^44 exp((x_i - m) / temperature)), a whole number, from a 64-bit exp;
//   the tokens in the order (x descending, index ascending);
//   kept: the first top_k of them; of these the shortest prefix whose sum of w
//   reaches top_p times the sum over the first top_k; of these the ones with
//   w >= min_p 2^44 (the first token always stays);
//   token = the first index, in the order of the vocabulary, at which the running
//   sum of the kept w exceeds floor(u * sum), logprob = ln(w / sum).
// Sums of whole numbers do not depend on their order, so neither do the
// borders between tokens: the histograms below may add in any order, and the
// result is the same for every split of a row.  A token below 2^-44 of the
// most likely one has weight 0.
//
// A cluster of up to eight CTAs takes a row; each holds its slice in shared
// memory, so the logits are read once.  All filters cut the same order, so each
// is found as a cut (key, ties): first by a histogram of kBins bins linear in
// (m - x) / temperature, then, inside the bin that holds the cut, by histograms
// over the ordered bit patterns until one value is left, whose ties are kept by
// index.  CTAs add their histograms through distributed shared memory.
#include "sample.cuh"

#include <cmath>

namespace kw8 {

namespace {

constexpr int kSampThreads = 512;
constexpr int kSampWarps = kSampThreads / 32;
constexpr int kBins = 1024;
constexpr float kBinsPerUnit = 32.f;  // bins per e-fold of the weight: the last one holds weights of 0
constexpr double kOne = 17592186044416.0;  // 2^44

using u64 = unsigned long long;

// Ordered like the value (no NaN, no -0).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// NaN -> -inf, -0 -> +0.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }

__device__ __forceinline__ float elem(const float* s, int i) { return s[i]; }
__device__ __forceinline__ float elem(const __nv_bfloat16* s, int i) { return __bfloat162float(s[i]); }
__device__ __forceinline__ void put(float* s, int i, float x) { s[i] = x; }
__device__ __forceinline__ void put(__nv_bfloat16* s, int i, float x) { s[i] = __float2bfloat16_rn(x); }

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// Shared state of a CTA besides its slice.
struct SampShared {
  u64 mass[kBins], mass_sum[kBins];
  uint32_t count[kBins], count_sum[kBins];
  u64 warp_a[kSampWarps];
  u64 pub[2];    // this CTA's value of a cluster-wide reduction (two: alternate)
  u64 cut[2];    // sum before the cut's bin
  uint32_t cut_bin, cut_count;
};

template <class Op>
__device__ __forceinline__ u64 block_reduce(u64 v, SampShared& sh, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_a[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = sh.warp_a[0];
  for (int i = 1; i < kSampWarps; ++i) r = op(r, sh.warp_a[i]);
  return r;
}

// Over all CTAs of the cluster; the same value in every thread.  `turn`
// alternates, so a value may be published while the last one is still read.
template <class Op>
__device__ __forceinline__ u64 cluster_reduce(u64 v, SampShared& sh, int ranks, int& turn, Op op) {
  v = block_reduce(v, sh, op);
  if (ranks == 1) return v;
  turn ^= 1;
  if (threadIdx.x == 0) sh.pub[turn] = v;
  cluster_sync_all();
  const uint32_t a = smem_u32(&sh.pub[turn]);
  u64 r = ld_cluster_u64(mapa_shared(a, 0));
  for (int i = 1; i < ranks; ++i) r = op(r, ld_cluster_u64(mapa_shared(a, static_cast<uint32_t>(i))));
  return r;
}

// Exclusive prefix of v over the cluster's threads, CTA by CTA; `total` is the sum.
__device__ __forceinline__ u64 cluster_prefix(u64 v, SampShared& sh, int ranks, int rank, int& turn, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) sh.warp_a[warp] = inc;
  __syncthreads();
  u64 base = 0, all = 0;
  for (int i = 0; i < kSampWarps; ++i) {
    if (i < warp) base += sh.warp_a[i];
    all += sh.warp_a[i];
  }
  total = all;
  if (ranks > 1) {
    turn ^= 1;
    if (threadIdx.x == 0) sh.pub[turn] = all;
    cluster_sync_all();
    const uint32_t a = smem_u32(&sh.pub[turn]);
    total = 0;
    for (int i = 0; i < ranks; ++i) {
      const u64 c = ld_cluster_u64(mapa_shared(a, static_cast<uint32_t>(i)));
      if (i < rank) base += c;
      total += c;
    }
  }
  return base + inc - v;
}

__device__ __forceinline__ void clear_hist(SampShared& sh) {
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSampThreads) {
    sh.mass[b] = 0;
    sh.count[b] = 0;
  }
  __syncthreads();
}

// Adds the CTAs' histograms: every CTA gets every bin.
__device__ __forceinline__ void sum_hist(SampShared& sh, int ranks) {
  if (ranks == 1) {
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kSampThreads) {
      sh.mass_sum[b] = sh.mass[b];
      sh.count_sum[b] = sh.count[b];
    }
    __syncthreads();
    return;
  }
  cluster_sync_all();
  for (int b = threadIdx.x; b < kBins; b += kSampThreads) {
    u64 m = 0;
    uint32_t c = 0;
    for (int i = 0; i < ranks; ++i) {
      m += ld_cluster_u64(mapa_shared(smem_u32(&sh.mass[b]), static_cast<uint32_t>(i)));
      c += ld_cluster_u32(mapa_shared(smem_u32(&sh.count[b]), static_cast<uint32_t>(i)));
    }
    sh.mass_sum[b] = m;
    sh.count_sum[b] = c;
  }
  cluster_sync_all();  // the histograms may be cleared again
}

struct Target {
  bool by_mass;
  u64 k;       // by count: the k-th
  double thr;  // by mass: the first whose running sum is not below thr
};

// Finds the bin in which the running sum, `before` in front of bin 0, reaches
// the target; leaves (bin, its count, the sum in front of it) in sh.
__device__ __forceinline__ void find_cut(SampShared& sh, const Target& t, u64 before) {
  constexpr int kPer = kBins / kSampThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 v[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int b = threadIdx.x * kPer + j;
    v[j] = t.by_mass ? sh.mass_sum[b] : sh.count_sum[b];
    sum += v[j];
  }
  u64 inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) sh.warp_a[warp] = inc;
  __syncthreads();
  u64 at = before + inc - sum;
  for (int i = 0; i < warp; ++i) at += sh.warp_a[i];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const u64 next = at + v[j];
    const bool here = t.by_mass ? (static_cast<double>(at) < t.thr && !(static_cast<double>(next) < t.thr))
                                : (at < t.k && next >= t.k);
    if (here) {
      sh.cut_bin = static_cast<uint32_t>(threadIdx.x * kPer + j);
      sh.cut_count = sh.count_sum[threadIdx.x * kPer + j];
      sh.cut[0] = at;
    }
    at = next;
  }
  __syncthreads();
}

template <class E>
__global__ void __launch_bounds__(kSampThreads)
    sample_kernel(const SampleArgs p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampShared& sh = *reinterpret_cast<SampShared*>(smem_raw);
  E* x = reinterpret_cast<E*>(smem_raw + sizeof(SampShared));
  uint32_t ranks_u;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks_u));
  const int ranks = static_cast<int>(ranks_u), rank = static_cast<int>(cluster_ctarank());
  const int64_t row = blockIdx.x / ranks;
  const int first = rank * p.slice;
  const int n = max(0, min(p.slice, p.V - first));
  const E* src = static_cast<const E*>(p.logits) + row * p.ld + first;
  int turn = 0;

  // The slice, and the row's first largest logit.
  u64 best = 0;  // (key, ~index): the largest value, of these the lowest index
  for (int i = threadIdx.x; i < n; i += kSampThreads) {
    const float v = clean(elem(src, i));
    put(x, i, v);
    best = max(best, (static_cast<u64>(order_key(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(first + i)));
  }
  best = cluster_reduce(best, sh, ranks, turn, [](u64 a, u64 b) { return a > b ? a : b; });
  const uint32_t top_key = static_cast<uint32_t>(best >> 32);
  const float top = key_value(top_key);
  const int top_index = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));

  const float temp = p.temperature ? p.temperature[row] : p.temperature0;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p0;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p0;
  const int32_t k = p.top_k ? p.top_k[row] : p.top_k0;

  if (top == -INFINITY || !(temp > 0.f) || !(top_p > 0.f) || !(min_p <= 1.f) || k == 1) {
    // No token at all, or the first most likely one.
    if (rank == 0 && threadIdx.x == 0) {
      const bool none = top == -INFINITY;
      p.token[row] = none ? -1 : top_index;
      if (p.logprob) p.logprob[row] = none ? -INFINITY : 0.f;
    }
    if (ranks > 1) cluster_sync_all();
    return;
  }

  const double inv_t = 1.0 / static_cast<double>(temp);
  const float bin_scale = fminf(kBinsPerUnit / temp, 1e30f);
  const auto weight = [&](float v) -> u64 {
    if (v == top) return static_cast<u64>(kOne);
    if (v == -INFINITY || top == INFINITY) return 0;
    return static_cast<u64>(exp((static_cast<double>(v) - static_cast<double>(top)) * inv_t) * kOne);
  };
  // Monotone in v: a subtraction, a product and a truncation.
  const auto bin_of = [&](float v) -> int {
    const float d = v == top ? 0.f : (top - v) * bin_scale;
    return static_cast<int>(fminf(d, static_cast<float>(kBins - 1)));
  };

  // The cut: tokens above cut_key stay, of those at it the first cut_ties.
  uint32_t cut_key = 0;
  uint32_t cut_ties = 0xffffffffu, cut_all = 0xffffffffu;  // kept, and present
  u64 ties_w = 0;

  // Inside bin `bin` (count elements, `before` the sum in front of it): the cut's key, its ties and how many of them stay.
  const auto refine = [&](const Target& t) {
    u64 before = sh.cut[0];
    uint32_t count = sh.cut_count;
    const int bin = static_cast<int>(sh.cut_bin);
    uint32_t lo = 0xffffffffu, hi = 0;
    for (int i = threadIdx.x; i < n; i += kSampThreads) {
      const float v = elem(x, i);
      if (bin_of(v) == bin) {
        const uint32_t key = order_key(v);
        lo = min(lo, key);
        hi = max(hi, key);
      }
    }
    lo = static_cast<uint32_t>(cluster_reduce(lo, sh, ranks, turn, [](u64 a, u64 b) { return a < b ? a : b; }));
    hi = static_cast<uint32_t>(cluster_reduce(hi, sh, ranks, turn, [](u64 a, u64 b) { return a > b ? a : b; }));
    while (lo != hi) {
      const int bits = 32 - __clz(static_cast<int>(hi - lo));
      const int shift = max(0, bits - 10);
      clear_hist(sh);
      for (int i = threadIdx.x; i < n; i += kSampThreads) {
        const float v = elem(x, i);
        const uint32_t key = order_key(v);
        if (key >= lo && key <= hi) {
          const uint32_t b = (hi - key) >> shift;
          atomicAdd(&sh.count[b], 1u);
          if (t.by_mass) atomicAdd(&sh.mass[b], weight(v));
        }
      }
      sum_hist(sh, ranks);
      find_cut(sh, t, before);
      before = sh.cut[0];
      count = sh.cut_count;
      const u64 b = sh.cut_bin;
      const u64 new_hi = hi - (b << shift);
      const u64 span = (1ull << shift) - 1;
      lo = new_hi - lo > span ? static_cast<uint32_t>(new_hi - span) : lo;
      hi = static_cast<uint32_t>(new_hi);
    }
    // One value left.
    const u64 w = weight(key_value(lo));
    uint32_t ties;
    if (t.by_mass) {
      uint32_t a = 1, b = count;  // the first always stays: `before` is below thr
      while (a < b) {
        const uint32_t mid = a + (b - a + 1) / 2;
        if (static_cast<double>(before + static_cast<u64>(mid - 1) * w) < t.thr) a = mid; else b = mid - 1;
      }
      ties = a;
    } else {
      ties = static_cast<uint32_t>(t.k - before);
    }
    if (lo > cut_key || (lo == cut_key && ties < cut_ties)) {
      cut_key = lo;
      cut_ties = ties;
      cut_all = count;
      ties_w = w;
    }
    __syncthreads();
  };

  if (k > 0 && k < p.V) {
    clear_hist(sh);
    for (int i = threadIdx.x; i < n; i += kSampThreads) atomicAdd(&sh.count[bin_of(elem(x, i))], 1u);
    sum_hist(sh, ranks);
    const Target t{false, static_cast<u64>(k), 0.0};
    find_cut(sh, t, 0);
    // In the last bin every weight is 0: whatever is kept of it is never drawn.
    if (sh.cut_bin < kBins - 1) refine(t);
    __syncthreads();
  }
  if (top_p < 1.f) {
    clear_hist(sh);
    u64 sum = 0;
    for (int i = threadIdx.x; i < n; i += kSampThreads) {
      const float v = elem(x, i);
      const int b = bin_of(v);
      if (b < kBins - 1 && order_key(v) >= cut_key) {
        const u64 w = weight(v);
        sum += w;
        atomicAdd(&sh.mass[b], w);
        atomicAdd(&sh.count[b], 1u);
      }
    }
    sum = cluster_reduce(sum, sh, ranks, turn, [](u64 a, u64 b) { return a + b; });
    if (cut_ties < cut_all) sum -= static_cast<u64>(cut_all - cut_ties) * ties_w;
    sum_hist(sh, ranks);
    const Target t{true, 0, static_cast<double>(top_p) * static_cast<double>(sum)};
    find_cut(sh, t, 0);
    refine(t);
  }

  // The draw.  Each thread owns a run of neighbouring tokens.
  const double least = static_cast<double>(min_p) * kOne;
  const int run = ((n + kSampThreads - 1) / kSampThreads) | 1;  // odd: no bank conflicts
  const int i0 = min(n, static_cast<int>(threadIdx.x) * run), i1 = min(n, i0 + run);
  u64 rank_of_tie = 0;
  if (cut_ties < cut_all) {
    u64 mine = 0, all;
    for (int i = i0; i < i1; ++i) mine += order_key(elem(x, i)) == cut_key;
    rank_of_tie = cluster_prefix(mine, sh, ranks, rank, turn, all);
  }
  const auto kept = [&](float v, u64& tie) -> u64 {
    const uint32_t key = order_key(v);
    if (key < cut_key) return 0;
    if (key == cut_key && tie++ >= cut_ties) return 0;
    const u64 w = weight(v);
    return static_cast<double>(w) >= least ? w : 0;
  };
  u64 mine = 0, tie = rank_of_tie, total;
  for (int i = i0; i < i1; ++i) mine += kept(elem(x, i), tie);
  u64 at = cluster_prefix(mine, sh, ranks, rank, turn, total);
  const double u = fmin(fmax(static_cast<double>(p.u[row]), 0.0), 1.0);
  const u64 goal = min(static_cast<u64>(u * static_cast<double>(total)), total - 1);
  if (at <= goal && goal < at + mine) {
    tie = rank_of_tie;
    for (int i = i0; i < i1; ++i) {
      const u64 w = kept(elem(x, i), tie);
      if (goal < at + w) {
        p.token[row] = first + i;
        if (p.logprob) p.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total)));
        break;
      }
      at += w;
    }
  }
  if (ranks > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <class E>
int launch_typed(SampleArgs p, int64_t B, cudaStream_t stream) {
  int dev = 0;
  KW8_CUDA_TRY(cudaGetDevice(&dev));
  static std::atomic<uint64_t> attr_set{0};
  const uint64_t bit = 1ull << (dev & 63);
  constexpr int kMaxSmem = 232448;
  if (!(attr_set.load() & bit)) {
    KW8_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    attr_set.fetch_or(bit);
  }
  // CTAs per row: eight while the rows leave SMs idle, then as few as hold a row with two CTAs on an SM.
  const int64_t fit = (110 * 1024 - static_cast<int64_t>(sizeof(SampShared))) / static_cast<int64_t>(sizeof(E));
  int64_t c = (p.V + fit - 1) / fit;
  c = std::max<int64_t>(c, std::min<int64_t>(8, (2 * 148 + B - 1) / B));
  c = std::min<int64_t>(std::min<int64_t>(c, 8), std::max<int64_t>(1, p.V / 1024));
  p.slice = static_cast<int>((p.V + c - 1) / c);
  const size_t smem = sizeof(SampShared) + static_cast<size_t>(p.slice) * sizeof(E);
  KW8_REQUIRE(smem <= static_cast<size_t>(kMaxSmem), KW8_ERR_UNSUPPORTED, "vocabulary of %d too large", p.V);
  KW8_REQUIRE(B * c < (1ll << 31), KW8_ERR_UNSUPPORTED, "too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B * c), 1, 1);
  cfg.blockDim = dim3(kSampThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(c);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c > 1 ? 1 : 0;
  KW8_CUDA_TRY(cudaLaunchKernelEx(&cfg, sample_kernel<E>, p));
  return KW8_OK;
}

}  // namespace

int launch_sample(const SampleArgs& args, int64_t B, int logits_dtype, cudaStream_t stream) {
  return logits_dtype == KW8_DT_F32 ? launch_typed<float>(args, B, stream)
                                    : launch_typed<__nv_bfloat16>(args, B, stream);
}

}  // namespace kw8
