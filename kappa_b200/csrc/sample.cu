// Token sampling: temperature, top-k, top-p and min-p, from given random numbers.
//
// Per row of logits x (NaN counts as -inf, +inf as the largest finite number),
// with m the largest:
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
// A cluster of up to sixteen CTAs takes a row; each holds its slice in shared
// memory, so the logits are read once (slices that leave no room for a second
// CTA on the SM are read from L1 and L2 again).  Every filter cuts the same order, so a
// histogram of kBins bins linear in (m - x) / temperature (a monotone function)
// finds the bin of each cut.  Then, with M the tokens down to that bin:
//   M <= kList: one CTA collects, sorts and finishes them (the usual settings);
//   else (flat rows, many ties, a wide nucleus): the cut is narrowed inside its
//   bin by histograms over the ordered bit patterns until one value is left,
//   whose ties are kept by index, and every CTA draws from its slice.  For top-p
//   alone the pass that sums the weights also lists the tokens of the bins that
//   the cut can lie in, and those steps go through them alone (64 x 151936 fp32,
//   top-p 0.9: 72 us, 110 through all tokens).
// CTAs add their histograms through distributed shared memory.
#include "sample.cuh"

#include "gemm_tc.cuh"

#include <cmath>

namespace kw8 {

namespace {

constexpr int kBins = 1024;
constexpr int kBinParts = 1024;    // positions told apart inside a bin where a top-p cut is bounded
constexpr float kBinSpan = 32.f;  // e-folds of the weight over all bins: the last one holds weights of 0
constexpr int kList = 1024;       // tokens that one CTA sorts
constexpr int kWindow = 2048;     // tokens around a top-p cut that a CTA lists
constexpr int kRanked = 256;      // up to here by counting, above by a sorting network
constexpr int kMaxRanks = 16;
constexpr int kMaxSmem = 232448;
constexpr double kOne = 17592186044416.0;  // 2^44
constexpr int kExpSteps = 64, kExpCopies = 8;  // table steps per octave of the exp (weight()), copies side by side

using u64 = unsigned long long;

// Ordered like the value (no NaN, no -0).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// NaN -> -inf, +inf -> the largest finite number of the type, -0 -> +0.
template <class E>
__device__ __forceinline__ float clean(float x) {
  constexpr float kMost = sizeof(E) == 4 ? 3.40282347e38f : 3.38953139e38f;
  return fminf(fmaxf(x, -INFINITY), kMost) + 0.0f;
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* s, int i, float x) { s[i] = x; }
__device__ __forceinline__ void put(__nv_bfloat16* s, int i, float x) { s[i] = __float2bfloat16_rn(x); }

// The 16 / sizeof(E) values of a vector and back.
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x);
  f[1] = __uint_as_float(v.y);
  f[2] = __uint_as_float(v.z);
  f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {  // the values are bf16 numbers: the upper halves
  return make_uint4(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x7632),
                    __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x7632),
                    __byte_perm(__float_as_uint(f[4]), __float_as_uint(f[5]), 0x7632),
                    __byte_perm(__float_as_uint(f[6]), __float_as_uint(f[7]), 0x7632));
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Shared state of a CTA besides its slice.
struct alignas(16) SampShared {
  // This CTA's histogram: a weight (45 bits) is added in pieces of 16, 16 and
  // 13 bits, each a 32-bit atomic (a CTA holds under 2^16 logits, so none
  // overflows); 64-bit atomics on shared memory are compare-and-swap loops.
  // The list of candidates takes the same memory.
  union {
    uint32_t mass[3][kBins];
    u64 list[kList];
  };
  uint32_t count[kBins];
  // The cluster's histogram; the collected list and its sort take the same memory.
  union {
    struct {
      u64 mass_sum[kBins];
      uint32_t count_sum[kBins];
    };
    u64 gathered[kList];
  };
  double exp_table[kExpSteps * kExpCopies];  // 2^(44 - i / kExpSteps)
  u64 warp_a[32];
  u64 warp_all[16][4];
  u64 pub[2][kMaxRanks][4];  // every CTA's values of a cluster-wide reduction (alternating)
  u64 cut_before;            // sum in front of the cut's bin
  uint32_t cut_bin, cut_count;
  uint32_t first_bin;           // of a top-p cut's window
  uint32_t windowed;            // its tokens in this CTA (entries of `window` while they fit)
  uint16_t window[kWindow];
  uint32_t listed;              // tokens of this CTA down to the cut (entries of `list` while they fit)
  uint32_t lists[kMaxRanks];    // every CTA's
};

__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 min64(u64 a, u64 b) { return a < b ? a : b; }
__device__ __forceinline__ u64 add64(u64 a, u64 b) { return a + b; }

// The least and the largest of some order keys, 0 for none, and two of these joined.
__device__ __forceinline__ u64 range(uint32_t lo, uint32_t hi) { return (static_cast<u64>(hi) << 32) | (~lo & 0xffffffffu); }
__device__ __forceinline__ u64 wider(u64 a, u64 b) {
  return (static_cast<u64>(max(static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b >> 32))) << 32) |
         max(static_cast<uint32_t>(a), static_cast<uint32_t>(b));
}

template <int kThreads>
struct Row {
  static constexpr int kWarps = kThreads / 32;
  static_assert(kWarps <= 16);
  SampShared& sh;
  const int ranks, rank;
  int turn = 0;

  __device__ Row(SampShared& s, int n, int r) : sh(s), ranks(n), rank(r) {}

  __device__ __forceinline__ void sync() {
    if (ranks > 1)
      cluster_sync_all();
    else
      __syncthreads();
  }

  template <class Op>
  __device__ __forceinline__ u64 block_reduce(u64 v, Op op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp_a[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.warp_a[(threadIdx.x & 31) % kWarps];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (o < kWarps) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }

  // Stores this CTA's values into every CTA's slot for it (thread r into CTA
  // r), and waits for all of them.  The slots alternate, so the last ones may
  // still be read meanwhile.
  template <int kN>
  __device__ __forceinline__ void publish(const u64 (&v)[kN]) {
    turn ^= 1;
    if (static_cast<int>(threadIdx.x) < ranks) {
      const uint32_t at = mapa_shared(smem_u32(sh.pub[turn][rank]), threadIdx.x);
#pragma unroll
      for (int j = 0; j < kN; ++j) st_cluster_u64(at + 8 * j, v[j]);
    }
    cluster_sync_all();
  }

  // Over all CTAs of the cluster; the same value in every thread.
  template <class Op>
  __device__ __forceinline__ u64 reduce(u64 v, Op op) {
    v = block_reduce(v, op);
    if (ranks == 1) return v;
    publish({v});
    u64 r = sh.pub[turn][0][0];
    for (int i = 1; i < ranks; ++i) r = op(r, sh.pub[turn][i][0]);
    return r;
  }

  // The same for a few sums and one range() at once.
  __device__ __forceinline__ void reduce_all(u64 (&v)[4]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
      for (int j = 0; j < 3; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], o);
      v[3] = wider(v[3], __shfl_xor_sync(0xffffffffu, v[3], o));
    }
    const int slot = threadIdx.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sh.warp_all[slot][j] = v[j];
    }
    __syncthreads();
    const auto add_up = [&](const auto& all, int n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = all[0][j];
      for (int i = 1; i < n; ++i) {
#pragma unroll
        for (int j = 0; j < 3; ++j) v[j] += all[i][j];
        v[3] = wider(v[3], all[i][3]);
      }
    };
    add_up(sh.warp_all, kWarps);
    if (ranks == 1) return;
    publish(v);
    add_up(sh.pub[turn], ranks);
  }

  // Exclusive prefix of v over this CTA's threads; `all` is their sum.
  __device__ __forceinline__ u64 block_prefix(u64 v, u64& all) {
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
    u64 base = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const u64 c = sh.warp_a[i];
      if (i < warp) base += c;
      all += c;
    }
    return base + inc - v;
  }

  // The same over the cluster's threads, CTA by CTA.
  __device__ __forceinline__ u64 prefix(u64 v, u64& total) {
    u64 all;
    u64 at = block_prefix(v, all);
    total = all;
    if (ranks > 1) {
      publish({all});
      total = 0;
      for (int i = 0; i < ranks; ++i) {
        const u64 c = sh.pub[turn][i][0];
        if (i < rank) at += c;
        total += c;
      }
    }
    return at;
  }

  __device__ __forceinline__ void clear(bool mass) {
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      if (mass)
        sh.mass[0][b] = sh.mass[1][b] = sh.mass[2][b] = 0;
      sh.count[b] = 0;
    }
    __syncthreads();
  }

  __device__ __forceinline__ void add_mass(int b, u64 w) {
    if (w == 0) return;
    atomicAdd(&sh.mass[0][b], static_cast<uint32_t>(w) & 0xFFFFu);
    atomicAdd(&sh.mass[1][b], static_cast<uint32_t>(w >> 16) & 0xFFFFu);
    atomicAdd(&sh.mass[2][b], static_cast<uint32_t>(w >> 32));
  }

  // Adds the CTAs' histograms: each sums its share of the bins, some threads
  // to a bin, and stores it into every CTA's copy.  Of the masses all three
  // pieces, or the first alone.
  __device__ __forceinline__ void sum(bool count, bool mass, bool pieces = true) {
    sync();
    const int share = (kBins + ranks - 1) / ranks;
    const int group = ranks >= 4 && kThreads >= 4 * share ? 4 : ranks >= 2 && kThreads >= 2 * share ? 2 : 1;
    const int part = static_cast<int>(threadIdx.x) % group;
    const int b0 = rank * share, b1 = min(kBins, b0 + share);
    // Whole warps go around together: the shuffles need them.
    for (int base = b0; base < b1; base += kThreads / group) {
      const int b = base + static_cast<int>(threadIdx.x) / group;
      const bool valid = b < b1;
      u64 m = 0;
      uint32_t c = 0;
      if (valid)
        for (int i = part; i < ranks; i += group) {
          const uint32_t r = static_cast<uint32_t>(i);
          if (count) c += ld_cluster_u32(mapa_shared(smem_u32(&sh.count[b]), r));
          if (mass) m += ld_cluster_u32(mapa_shared(smem_u32(&sh.mass[0][b]), r));
          if (mass && pieces)
            m += (static_cast<u64>(ld_cluster_u32(mapa_shared(smem_u32(&sh.mass[1][b]), r))) << 16) +
                 (static_cast<u64>(ld_cluster_u32(mapa_shared(smem_u32(&sh.mass[2][b]), r))) << 32);
        }
      for (int o = 1; o < group; o <<= 1) {
        c += __shfl_xor_sync(0xffffffffu, c, o);
        m += __shfl_xor_sync(0xffffffffu, m, o);
      }
      if (valid)
        for (int i = part; i < ranks; i += group) {
          const uint32_t r = static_cast<uint32_t>(i);
          st_cluster_u32(mapa_shared(smem_u32(&sh.count_sum[b]), r), c);
          if (mass) st_cluster_u64(mapa_shared(smem_u32(&sh.mass_sum[b]), r), m);
        }
    }
    sync();  // the sums are complete, and the histograms may be cleared again
  }

  // Finds the bin in which the running sum (of the counts: up to k; of the
  // masses: up to thr), `before` in front of bin 0, reaches its goal, and leaves
  // it in sh: the bin, its count and the sum in front of it.
  __device__ __forceinline__ void find_cut(bool by_mass, u64 k, double thr, u64 before) {
    constexpr int kPer = kBins / kThreads;
    u64 v[kPer], s = 0, all;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int b = threadIdx.x * kPer + j;
      v[j] = by_mass ? sh.mass_sum[b] : sh.count_sum[b];
      s += v[j];
    }
    u64 at = before + block_prefix(s, all);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const u64 next = at + v[j];
      const bool here = by_mass ? (static_cast<double>(at) < thr && !(static_cast<double>(next) < thr))
                                : (at < k && next >= k);
      if (here) {
        sh.cut_bin = static_cast<uint32_t>(threadIdx.x * kPer + j);
        sh.cut_count = sh.count_sum[threadIdx.x * kPer + j];
        sh.cut_before = at;
      }
      at = next;
    }
    __syncthreads();
  }

  // From the counts, and where `fine` from the positions inside the bins
  // (count_positions()): the bins between which the top_p cut must lie.  The
  // exponential is convex: with s the bins' span, the weights of bin b's c tokens,
  // whose positions in it have the sum S, add up to at most e^(-b s) (c - S (1 - e^-s))
  // (the chord) and to at least e^(-(b + 1/2) s) (c - (S - c / 2) s) (the tangent in
  // the middle), 0.024% less; without S 3% lie between its ends.  Besides, positions
  // are rounded down to 2^-10 bins and weights to whole numbers, and 3 roundings of
  // 2^-24 move a position by at most 0.0002 bins.  The sum down to the cut is
  // compared with top_p of all and the sum behind it with 1 - top_p of all, which
  // is the sharper one near 1 (64 x 151936 fp32, top-p 0.9999: 72 us, 165 without).
  // sh.first_bin, sh.cut_bin: raised to the first bin that the cut can lie in, and
  // lowered to the first that it cannot lie behind.
  __device__ __forceinline__ void bound_cut(double top_p, bool fine) {
    constexpr int kPer = kBins / kThreads;
    constexpr double kSpan = static_cast<double>(kBinSpan) / (kBins - 1), kMoved = 0.0005;
    constexpr double kStep = kSpan * (1 - kSpan / 2);                          // at most 1 - e^-s
    constexpr double kHalf = 1 - kSpan / 2 * (1 - kSpan / 4 * (1 - kSpan / 6));  // at most e^(-s / 2)
    u64 lo[kPer], hi[kPer], slo = 0, shi = 0, all_lo, all_hi;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int b = threadIdx.x * kPer + j;
      const double c = sh.count_sum[b], S = fine ? static_cast<double>(sh.mass_sum[b]) * (1.0 / kBinParts) : 0.0;
      const double w = kOne * exp(-(b - kMoved) * kSpan);
      const double most = c - S * kStep;
      const double least = kHalf * (c - ((fine ? S + c * (1.0 / kBinParts) : c) + c * (2 * kMoved - 0.5)) * kSpan);
      lo[j] = static_cast<u64>(fmax(w * least * (1 - 1e-12) - c, 0.0));
      hi[j] = static_cast<u64>(ceil(w * most * (1 + 1e-12)));
      slo += lo[j];
      shi += hi[j];
    }
    u64 at_lo = block_prefix(slo, all_lo), at_hi = block_prefix(shi, all_hi);
    const double total_lo = static_cast<double>(all_lo), total_hi = static_cast<double>(all_hi);
    const double least = top_p * total_lo * (1 - 1e-12), most = top_p * total_hi * (1 + 1e-12);
    // (1e-14 of all: the roundings where the exact sums are compared with top_p of them.)
    const double tail_least = (1 - top_p) * total_lo * (1 - 1e-12) - 1e-14 * total_hi;
    const double tail_most = (1 - top_p) * total_hi * (1 + 1e-12) + 1e-14 * total_hi;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const uint32_t b = threadIdx.x * kPer + j;
      const double from_lo = static_cast<double>(all_lo - at_lo), behind_lo = static_cast<double>(all_lo - at_lo - lo[j]);
      const double from_hi = static_cast<double>(all_hi - at_hi), behind_hi = static_cast<double>(all_hi - at_hi - hi[j]);
      if ((static_cast<double>(at_hi) < least && !(static_cast<double>(at_hi + hi[j]) < least)) ||
          (from_lo > tail_most && !(behind_lo > tail_most)))
        atomicMax(&sh.first_bin, b);
      if ((static_cast<double>(at_lo) < most && !(static_cast<double>(at_lo + lo[j]) < most)) ||
          (from_hi > tail_least && !(behind_hi > tail_least)))
        atomicMin(&sh.cut_bin, b);
      at_lo += lo[j];
      at_hi += hi[j];
    }
    __syncthreads();
  }

  // Tokens in the bins up to and with `bin`.
  __device__ __forceinline__ u64 count_to(int bin) {
    u64 c = 0;
    for (int b = threadIdx.x; b <= bin; b += kThreads) c += sh.count_sum[b];
    return block_reduce(c, [](u64 a, u64 b) { return a + b; });
  }

  // a[0 .. size) into descending order; size a power of two.
  __device__ __forceinline__ void sort(u64* a, int size) {
    for (int len = 2; len <= size; len <<= 1)
      for (int step = len >> 1; step > 0; step >>= 1) {
        for (int i = threadIdx.x; i < size / 2; i += kThreads) {
          const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
          const u64 p = a[lo], q = a[hi];
          if ((p < q) == ((lo & len) == 0)) {
            a[lo] = q;
            a[hi] = p;
          }
        }
        __syncthreads();
      }
  }
};

// What is known at the launch of every row's filters.  In a kernel of their own
// they lose no registers and instructions to the other paths (64 x 151936 fp32,
// top-k 50: 24.9 us, 28 in the one for any; 1 x 151936 bf16 top-p 0.9: 24.7
// against 25.3; 256 x 32000 fp32 without filters: 24.1 against 25.7).
enum Filters { kNone, kTopK, kNoTopK, kAny };

template <class E, int kThreads, bool kStaged, Filters kFilters>
__global__ void __launch_bounds__(kThreads, 2)
    sample_kernel(const SampleArgs p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampShared& sh = *reinterpret_cast<SampShared*>(smem_raw);
  uint32_t ranks_u;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks_u));
  const int ranks = static_cast<int>(ranks_u), rank = ranks > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  Row<kThreads> R(sh, ranks, rank);
  const int tid = static_cast<int>(threadIdx.x);
  const int64_t row = blockIdx.x / ranks;
  const int first = rank * p.slice;
  const int n = max(0, min(p.slice, p.V - first));
  const E* src = static_cast<const E*>(p.logits) + row * p.ld + (n > 0 ? first : 0);

  // The first exchange below stores into the other CTAs, which must have started: their slices' loads lie
  // between the two halves of this barrier.
  if (ranks > 1) cluster_arrive_relaxed();

  const float temp = p.temperature ? p.temperature[row] : p.temperature0;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p0;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p0;
  const int32_t k = p.top_k ? p.top_k[row] : p.top_k0;
  for (int i = tid; i < kExpSteps * kExpCopies; i += kThreads)
    sh.exp_table[i] = exp2(44.0 - (i / kExpCopies) * (1.0 / kExpSteps));
  if (tid == 0) sh.listed = 0;

  // The row's first largest logit.  The slice is read in whole vectors, with
  // single values at its ends; kStaged: into shared memory, at the alignment that
  // it has in global memory, else later passes find it in L1 and L2.
  constexpr int kVec = 16 / sizeof(E);
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(E));
  const uint4* const gsrc = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src) & ~static_cast<uintptr_t>(15));
  E* const aligned = reinterpret_cast<E*>(smem_raw + sizeof(SampShared));
  const int v0 = (lead + kVec - 1) / kVec, v1 = (lead + n) / kVec;  // whole vectors
  const int head = min(n, v0 * kVec - lead), tail = max(head, v1 * kVec - lead);
  float best = -INFINITY;
  int best_at = -1;  // none above -inf yet
  {
    constexpr int kUnroll = 6;
    const auto single = [&](int i) {
      const float f = clean<E>(to_float(src[i]));
      if constexpr (kStaged) put(aligned + lead, i, f);
      if (f > best) best = f, best_at = i;
    };
    if (tid < head) single(tid);
    for (int base = v0 + tid; base < v1; base += kUnroll * kThreads) {
      uint4 v[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
        if (base + j * kThreads < v1) v[j] = __ldg(gsrc + base + j * kThreads);
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
        if (base + j * kThreads < v1) {
          float f[kVec];
          unpack(v[j], f);
          const int i = (base + j * kThreads) * kVec;
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            f[e] = clean<E>(f[e]);
            if (f[e] > best) best = f[e], best_at = i + e - lead;
          }
          if constexpr (kStaged) *reinterpret_cast<uint4*>(aligned + i) = pack(f);
        }
    }
    if (tail + tid < n) single(tail + tid);
  }
  // Token i of the slice.
  const E* const x = kStaged ? aligned + lead : src;
  const auto elem = [x](int i) -> float {
    if constexpr (kStaged)
      return to_float(x[i]);
    else
      return clean<E>(to_float(__ldg(x + i)));
  };
  if (ranks > 1) {
    __syncwarp();
    cluster_wait();
  }
  // (key, ~index): the largest value, of equals the lowest index.
  const u64 best_all = R.reduce(
      best_at < 0 ? 0 : (static_cast<u64>(order_key(best)) << 32) | (0xffffffffu - static_cast<uint32_t>(first + best_at)),
      max64);
  if (best_all == 0 || !(temp > 0.f) || !(top_p > 0.f) || !(min_p <= 1.f) || k == 1) {
    // No token at all, or the first most likely one.
    if (rank == 0 && tid == 0) {
      p.token[row] = best_all == 0 ? -1 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best_all));
      if (p.logprob) p.logprob[row] = best_all == 0 ? -INFINITY : 0.f;
    }
    if (ranks > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
    return;
  }
  const float top = key_value(static_cast<uint32_t>(best_all >> 32));

  // floor(2^44 exp(-d / temperature)), d = m - v, by Tang's table-driven
  // exponential: d in steps of ln2 / 64, 2^(44 - n/64) from the table (the octaves
  // subtracted from the exponent), the rest (at most ln2 / 128) by its series to
  // the 5th power (error below 4e-17), rounded down by adding 2^52.  No branches,
  // so that several run at once; eight copies of the table, so that few lanes
  // meet in a bank.  Where every token is weighed, the 64-bit pipe and the issue
  // slots bound the kernel: 13 64-bit operations and about as many others, 10.5
  // cycles of an SM per warp (with shifts and selects of 64-bit words instead of
  // the additions 13.6), whatever the unrolling.
  const double top_d = static_cast<double>(top);
  const double per_step = kExpSteps * 1.4426950408889634 / static_cast<double>(temp);
  const uint32_t d_end = static_cast<uint32_t>(__double2hiint(46 * 0.6931471805599453 * static_cast<double>(temp)));
  const double* const table = sh.exp_table + (tid & (kExpCopies - 1));
  const auto weight = [&](float v) -> u64 {
    constexpr double h = -0.6931471805599453 / kExpSteps;
    const double d = top_d - static_cast<double>(v);
    const double z = fma(d, per_step, 6755399441055744.0);  // 1.5 * 2^52: the low word is the nearest integer
    const double f = fma(d, per_step, 6755399441055744.0 - z);
    const int steps = __double2loint(z);
    double e = fma(f, h * h * h * h * h / 120, h * h * h * h / 24);
    e = fma(e, f, h * h * h / 6);
    e = fma(e, f, h * h / 2);
    e = fma(e, f, h);
    e = fma(e, f, 1.0);
    e *= table[(steps & (kExpSteps - 1)) * kExpCopies];
    // From 46 octaves on, and for -inf, nothing is left.
    const bool far = static_cast<uint32_t>(__double2hiint(d)) >= d_end;
    const int hi = far ? 0 : __double2hiint(e) - ((steps >> 6) << 20);
    e = __dadd_rd(__hiloint2double(hi, __double2loint(e)), 4503599627370496.0);
    return static_cast<u64>(__double_as_longlong(e)) & 0xFFFFFFFFFFFFFull;
  };
  // Monotone in v: a subtraction, a product cut to [0, 1], a product rounded
  // down (by adding 2^23).
  // At temperatures below 1 / (32 kMostScale) the bins are wider than that; the last one begins further than
  // kBinSpan e-folds from the maximum, so its weights are 0 all the same.
  constexpr float kMostScale = 1e30f;
  const float bin_scale = fminf(1.f / (kBinSpan * temp), kMostScale);
  const auto bin_of = [&](float v) -> int {
    const float d = __saturatef((top - v) * bin_scale);
    return static_cast<int>(__float_as_uint(__fmaf_rz(d, static_cast<float>(kBins - 1), 8388608.f)) & (kBins - 1));
  };

  // The logit at bin position `at`, two steps of the format up or down, which
  // covers its rounding: tokens above upper(b - 0.5) lie in bins below b, tokens of
  // the bins up to b not below lower(b + 1.5).
  const auto edge_key = [&](float at) { return order_key(top - at / static_cast<float>(kBins - 1) / bin_scale + 0.0f); };
  const auto upper = [&](float at) { return key_value(min(edge_key(at) + 2, 0xFF800000u)); };
  const auto lower = [&](float at) { return key_value(max(edge_key(at), 0x00800001u) - 2); };

  const bool use_k = kFilters == kTopK || (kFilters == kAny && k > 0 && k < p.V);
  const bool use_p = kFilters != kNone && top_p < 1.f, use_m = kFilters != kNone && min_p > 0.f;
  // w >= min_p 2^44 in whole numbers (the product is exact).
  const u64 least = use_m ? static_cast<u64>(ceil(static_cast<double>(min_p) * kOne)) : 0;
  const auto enough = [&](u64 w) { return !use_m || w >= least; };
  const double u = fmin(fmax(static_cast<double>(p.u[row]), 0.0), 1.0);

  // For sums in the order of the vocabulary each thread owns a run of
  // neighbouring tokens.
  const int run_len = ((n + kThreads - 1) / kThreads) | 1;  // odd: no bank conflicts
  const int i0 = min(n, tid * run_len), i1 = min(n, i0 + run_len);
  const auto over_run = [&](auto&& f) {
#pragma unroll 4
    for (int i = i0; i < i1; ++i) f(elem(i), i);
  };
  // Sum of this thread's tokens above run_top, in front of the window in which a
  // mass cut lies: certain to stay, and summed already.
  u64 run_sum = 0;
  float run_top = INFINITY;

  // Whether sh.window lists that window's tokens, and every one of the cluster's
  // CTAs had room for its own.
  bool listed = false;
  u64 window_front = 0, window_count = 0, window_range = 0;  // the sum in front of it, its tokens, their keys

  // The key of a cut: a bf16 number's upper half is enough.
  const auto cut_key_of = [](float v) { return sizeof(E) == 2 ? order_key(v) >> 16 : order_key(v); };
  const auto cut_value = [](uint32_t key) {
    return key_value(sizeof(E) == 2 ? (key << 16) | (key & 0x8000u ? 0u : 0xFFFFu) : key);
  };

  // The cut of the general path: tokens above cut_key stay, of those at it the first cut_ties.
  uint32_t cut_key = 0;
  uint32_t cut_ties = 0xffffffffu, cut_all = 0xffffffffu;  // kept, and present

  // f(value, index) for every token of the slice, in no order; go() ends it.
  const auto for_each = [&](auto&& f, auto&& go) {
    if (tid < head) f(elem(tid), tid);
    if (tail + tid < n) f(elem(tail + tid), tail + tid);
    constexpr int kAtOnce = kStaged ? 1 : 4;  // vectors in flight
    for (int b = v0 + tid; b < v1 && go(); b += kAtOnce * kThreads) {
      uint4 v[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (b + j * kThreads < v1) v[j] = kStaged ? reinterpret_cast<const uint4*>(aligned)[b] : __ldg(gsrc + b + j * kThreads);
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (b + j * kThreads < v1) {
          float fv[kVec];
          unpack(v[j], fv);
          const int i = (b + j * kThreads) * kVec - lead;
#pragma unroll
          for (int e = 0; e < kVec; ++e) f(kStaged ? fv[e] : clean<E>(fv[e]), i + e);
        }
    }
  };
  const auto always = [] { return true; };
  // The same for the tokens that a cut can lie at.
  const auto for_window = [&](auto&& f) {
    if (listed) {
      for (int i = tid; i < static_cast<int>(sh.windowed); i += kThreads) f(elem(sh.window[i]), sh.window[i]);
    } else {
      for_each(f, always);
    }
  };
  const auto count_all = [&] {
    for_each([&](float v, int) { atomicAdd(&sh.count[bin_of(v)], 1u); }, always);
  };
  // And the sums of the positions inside the bins, in mass[0] (under 2^16 tokens of
  // 10 bits).  The bin is bin_of's: both round the same product down.
  const auto count_positions = [&] {
    for_each(
        [&](float v, int) {
          const float d = __saturatef((top - v) * bin_scale);
          const uint32_t at = __float_as_uint(__fmaf_rz(d, static_cast<float>((kBins - 1) * kBinParts), 8388608.f)) & (kBins * kBinParts - 1);
          atomicAdd(&sh.count[at / kBinParts], 1u);
          atomicAdd(&sh.mass[0][at / kBinParts], at % kBinParts);
        },
        always);
  };
  if (use_k || use_p || use_m) {
    // Counts find the bin of a top-k cut, and bound a top-p cut, with the positions
    // inside the bins to a window of a bin or two (not worth their sums where min_p
    // bounds it besides: 16 x 262144 bf16, top-p 0.9, min-p 0.02: 37 us, 44 with them).
    const bool mass = use_p && !use_k, fine = mass && !use_m;
    // When at least top_k threads hold a token, the top_k-th largest of the
    // threads' own largest logits already bounds the cut (that many tokens are
    // not below it), at one addition per thread instead of one per token.
    int last = kBins - 1;  // nothing kept lies behind this bin
    double thr = 0.0;
    const bool by_threads = use_k && k <= kThreads * ranks / 2 && p.V >= kThreads * ranks;
    if (use_k || use_p) {
      R.clear(fine);
      if (fine)
        count_positions();
      else if (!by_threads)
        count_all();
      else if (best_at >= 0)
        atomicAdd(&sh.count[bin_of(best)], 1u);
      R.sum(true, fine, false);
      // Fewer threads than top_k above -inf: no bound, every token may be kept.
      sh.cut_bin = kBins - 1;
      sh.first_bin = 0;
      __syncthreads();
      if (use_k) {
        R.find_cut(false, static_cast<u64>(k), 0.0, 0);
      } else if (bin_scale < kMostScale && bin_scale > 2e-38f) {  // bins of the width that bound_cut() takes them for:
        // wider at the most, and below 2e-38 the scale loses bits, and is 0 in the end
        R.bound_cut(static_cast<double>(top_p), fine);
        if (sh.first_bin > 0) run_top = upper(static_cast<float>(sh.first_bin) - 0.5f);
      }
      last = static_cast<int>(sh.cut_bin);
    }
    // w >= min_p 2^44 means (m - x) / temperature <= -ln min_p; two bins cover
    // the roundings.  (With top-k and top-p the list has to hold all top_k.)
    if (use_m && !(use_k && use_p))
      last = min(last, static_cast<int>(fminf(-logf(min_p) * ((kBins - 1) / kBinSpan), static_cast<float>(kBins))) + 2);

    bool window = false;
    if (mass) {
      // All weights once: their sum, and where the list will not do (it reaches up
      // to two bins further, see below) this thread's part of it in front of the
      // window, and the tokens of the window, if there is room for them.
      if (tid == 0) sh.windowed = 0;
      window = R.count_to(min(last + 2, kBins - 1)) > kList;
      u64 sum = 0;
      if (!window) {
        over_run([&](float v, int) { sum += weight(v); });
        sum = R.reduce(sum, add64);
      } else {
        const int window_end = static_cast<int>(sh.cut_bin);
        const float window_low = lower(static_cast<float>(window_end) + 1.5f);
        uint32_t lo = 0xffffffffu, hi = 0;
        over_run([&](float v, int i) {
          const u64 w = weight(v);
          sum += w;
          run_sum += v > run_top ? w : 0;
          if (v <= run_top && v >= window_low) {
            const uint32_t at = atomicAdd(&sh.windowed, 1u);
            if (at < kWindow) sh.window[at] = static_cast<uint16_t>(i);
          }
        });
        __syncthreads();
        for (int i = tid; i < min(static_cast<int>(sh.windowed), kWindow); i += kThreads) {
          const uint32_t key = cut_key_of(elem(sh.window[i]));
          lo = min(lo, key);
          hi = max(hi, key);
        }
        const u64 room = sh.windowed <= kWindow ? 0 : 1ull << 32;
        u64 all[4] = {sum, run_sum, tid == 0 ? sh.windowed + room : 0, range(lo, hi)};
        R.reduce_all(all);
        sum = all[0];
        thr = static_cast<double>(top_p) * static_cast<double>(sum);
        window_front = all[1];
        window_count = all[2];
        window_range = all[3];
        listed = window_count < (1ull << 32);
        if (!listed) {  // the bin of the cut first
          R.clear(true);
          for_each(
              [&](float v, int) {
                if (v <= run_top && v >= window_low) {
                  const int b = bin_of(v);
                  if (b <= window_end) R.add_mass(b, weight(v));
                }
              },
              always);
          R.sum(false, true);
          R.find_cut(true, 0, thr, window_front);
        }
      }
      thr = static_cast<double>(top_p) * static_cast<double>(sum);
    }

    // Collect the tokens down to bin `last` as (key, ~index), as far as they fit.
    // The bin as a bound on the logit (tokens of the two bins behind do no harm).
    if (!window) {
      const int behind = min(last + 2, kBins - 1);
      const float bound = last < kBins - 1 ? lower(static_cast<float>(last) + 1.5f) : -INFINITY;
      for_each(
          [&](float v, int i) {
            if (v >= bound && bin_of(v) <= behind) {
              const uint32_t at = atomicAdd(&sh.listed, 1u);
              if (at < kList) sh.list[at] = (static_cast<u64>(order_key(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(first + i));
            }
          },
          [&] { return *static_cast<volatile uint32_t*>(&sh.listed) <= kList; });  // not too many already
    } else if (tid == 0) {
      sh.listed = kList + 1;
    }
    __syncthreads();
    if (ranks > 1) {
      if (tid < ranks) st_cluster_u32(mapa_shared(smem_u32(&sh.lists[rank]), static_cast<uint32_t>(tid)), sh.listed);
      cluster_sync_all();
    }
    int M = 0, my_place = 0;
    if (ranks > 1)
      for (int r = 0; r < ranks; ++r) M += static_cast<int>(sh.lists[r]);
    else
      M = static_cast<int>(sh.listed);

    if (M <= kList) {
      // CTA 0 finishes.  Each CTA's list goes behind the ones before it.
      if (ranks > 1) {
        for (int r = 0; r < rank; ++r) my_place += static_cast<int>(sh.lists[r]);
        for (int i = tid; i < static_cast<int>(sh.lists[rank]); i += kThreads)
          st_cluster_u64(mapa_shared(smem_u32(&sh.gathered[my_place + i]), 0), sh.list[i]);
        cluster_sync_all();
        if (rank != 0) return;
      } else {
        for (int i = tid; i < M; i += kThreads) sh.gathered[i] = sh.list[i];
        __syncthreads();
      }
      const int limit = use_k ? min(M, k) : M;
      if (M <= kRanked) {
        // Each token's place: how many come before it.  kGroup threads per token.
        constexpr int kGroup = kThreads / kRanked;
        const int i = tid / kGroup, part = tid % kGroup;
        u64* const weights = sh.list;
        const u64 e = i < M ? sh.gathered[i] : 0;
        int place = 0;
        for (int j = part; j < M; j += kGroup) place += sh.gathered[j] > e;
#pragma unroll
        for (int o = 1; o < kGroup; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
        const bool in = i < M && place < limit;
        const u64 w0 = in ? weight(key_value(static_cast<uint32_t>(e >> 32))) : 0;
        if (part == 0 && i < M) weights[place] = w0;
        __syncthreads();
        u64 before, total;  // running sum in front of place `tid`
        const u64 wp = tid < M ? weights[tid] : 0;
        before = R.block_prefix(wp, total);
        const double goal_p = mass ? thr : static_cast<double>(top_p) * static_cast<double>(total);
        const bool keep = tid == 0 || (tid < limit && (!use_p || static_cast<double>(before) < goal_p) &&
                                       enough(wp));
        // The kept ones are the first places: their number, and their sum.
        const u64 both = R.block_reduce(keep ? before + wp : 0, max64);
        total = both;
        const int kept = static_cast<int>(R.block_reduce(keep ? tid + 1 : 0, max64));
        // In the order of the vocabulary: the sum of the kept ones with a lower index.
        const u64 w = in && place < kept ? w0 : 0;
        __syncthreads();
        if (part == 0 && i < M) weights[i] = w;
        __syncthreads();
        const uint32_t id = static_cast<uint32_t>(e);  // ~index: higher means earlier
        u64 run = 0;
        for (int j = part; j < M; j += kGroup) run += static_cast<uint32_t>(sh.gathered[j]) > id ? weights[j] : 0;
#pragma unroll
        for (int o = 1; o < kGroup; o <<= 1) run += __shfl_xor_sync(0xffffffffu, run, o);
        const u64 goal = min64(static_cast<u64>(u * static_cast<double>(total)), total - 1);
        if (part == 0 && w != 0 && run <= goal && goal < run + w) {
          p.token[row] = static_cast<int32_t>(0xffffffffu - id);
          if (p.logprob) p.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total)));
        }
        return;
      }
      int size = 64;
      while (size < M) size *= 2;
      for (int i = M + tid; i < size; i += kThreads) sh.gathered[i] = 0;
      __syncthreads();
      R.sort(sh.gathered, size);
      // Thread t owns the kPer places from t * kPer on.
      constexpr int kPer = (kList + kThreads - 1) / kThreads;
      u64 e[kPer], w[kPer], mine = 0, total;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        e[j] = i < limit ? sh.gathered[i] : 0;
        w[j] = i < limit ? weight(key_value(static_cast<uint32_t>(e[j] >> 32))) : 0;
        mine += w[j];
      }
      u64 before = R.block_prefix(mine, total);
      const double goal_p = mass ? thr : static_cast<double>(top_p) * static_cast<double>(total);
      u64 kept = 0;
      mine = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        const bool keep =
            i == 0 || (i < limit && (!use_p || static_cast<double>(before) < goal_p) && enough(w[j]));
        before += w[j];
        if (!keep) w[j] = 0;
        kept += keep;
        mine += w[j];
      }
      kept = R.block_reduce(kept, add64);  // the first `kept` places
      total = R.block_reduce(mine, add64);
      // In the order of the vocabulary: descending ~index, with the place; weights go to `list`.
      u64* const weights = sh.list;
      size = 64;
      while (size < static_cast<int>(kept)) size *= 2;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        if (i < size) {
          sh.gathered[i] = i < static_cast<int>(kept) ? (e[j] << 32) | static_cast<uint32_t>(i) : 0;
          weights[i] = w[j];
        }
      }
      __syncthreads();
      R.sort(sh.gathered, size);
      mine = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = tid * kPer + j;
        e[j] = i < static_cast<int>(kept) ? sh.gathered[i] : 0;
        w[j] = i < static_cast<int>(kept) ? weights[static_cast<uint32_t>(e[j])] : 0;
        mine += w[j];
      }
      u64 all;
      u64 run = R.block_prefix(mine, all);
      const u64 goal = min64(static_cast<u64>(u * static_cast<double>(total)), total - 1);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (run <= goal && goal < run + w[j]) {
          p.token[row] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e[j] >> 32));
          if (p.logprob) p.logprob[row] = static_cast<float>(log(static_cast<double>(w[j]) / static_cast<double>(total)));
        }
        run += w[j];
      }
      return;
    }

    // The general path.  Inside the bin that sh's cut is in: the cut's key, its ties and how many of them stay.
    u64 ties_w = 0;
    const auto refine = [&](bool by_mass, u64 goal_k, double goal_p) {
      u64 before = window_front, count = window_count, keys = window_range;
      if (!listed) {
        before = sh.cut_before;
        const int bin = static_cast<int>(sh.cut_bin);
        const float above = bin > 0 ? upper(static_cast<float>(bin) - 0.5f) : INFINITY;
        const float below = bin < kBins - 1 ? lower(static_cast<float>(bin) + 1.5f) : -INFINITY;
        uint32_t lo = 0xffffffffu, hi = 0, mine = 0;
        for_each(
            [&](float v, int) {
              if (v <= above && v >= below && bin_of(v) == bin) {
                lo = min(lo, cut_key_of(v));
                hi = max(hi, cut_key_of(v));
                ++mine;
              }
            },
            always);
        u64 all[4] = {mine, 0, 0, range(lo, hi)};
        R.reduce_all(all);
        count = all[0];
        keys = all[3];
      }
      u64 lo = ~static_cast<uint32_t>(keys), hi = keys >> 32;
      // Each level leaves 2^10 times fewer values: four at most.
      for (int level = 0; level < 4 && lo != hi; ++level) {
        const int bits = 32 - __clz(static_cast<int>(hi - lo));
        const int shift = max(0, bits - 10);
        R.clear(by_mass);
        const float least_v = cut_value(static_cast<uint32_t>(lo)), most_v = cut_value(static_cast<uint32_t>(hi));
        for_window([&](float v, int) {
          if (v >= least_v && v <= most_v) {
            const int b = static_cast<int>((hi - cut_key_of(v)) >> shift) & (kBins - 1);
            atomicAdd(&sh.count[b], 1u);
            if (by_mass) R.add_mass(b, weight(v));
          }
        });
        R.sum(true, by_mass);
        R.find_cut(by_mass, goal_k, goal_p, before);
        before = sh.cut_before;
        count = sh.cut_count;
        hi -= static_cast<u64>(sh.cut_bin) << shift;
        const u64 span = (1ull << shift) - 1;
        if (hi - lo > span) lo = hi - span;
      }
      // One value left.
      const uint32_t key = static_cast<uint32_t>(lo);
      const u64 w = weight(cut_value(key));
      uint32_t ties;
      if (by_mass) {
        uint32_t a = 1, b = static_cast<uint32_t>(count);  // the first always stays: `before` is below the goal
        while (a < b) {
          const uint32_t mid = a + (b - a + 1) / 2;
          if (static_cast<double>(before + static_cast<u64>(mid - 1) * w) < goal_p) a = mid; else b = mid - 1;
        }
        ties = a;
      } else {
        ties = static_cast<uint32_t>(goal_k - before);
      }
      if (key > cut_key || (key == cut_key && ties < cut_ties)) {
        cut_key = key;
        cut_ties = ties;
        cut_all = static_cast<uint32_t>(count);
        ties_w = w;
      }
      __syncthreads();
    };

    if (by_threads) {
      R.clear(false);
      count_all();
      R.sum(true, false);
      R.find_cut(false, static_cast<u64>(k), 0.0, 0);
    }
    // In the last bin every weight is 0: whatever is kept of it is never drawn.
    if (listed || ((use_k || use_p) && sh.cut_bin < kBins - 1)) refine(mass, static_cast<u64>(k), thr);
    if (use_k && use_p) {
      R.clear(true);
      u64 s = 0;
      const float cut_v = cut_key == 0 ? -INFINITY : cut_value(cut_key);
      for_each(
          [&](float v, int) {
            if (v >= cut_v) {
              const u64 w = weight(v);
              s += w;
              R.add_mass(bin_of(v), w);
            }
          },
          always);
      s = R.reduce(s, add64);
      if (cut_ties < cut_all) s -= static_cast<u64>(cut_all - cut_ties) * ties_w;
      R.sum(false, true);
      const double goal = static_cast<double>(top_p) * static_cast<double>(s);
      R.find_cut(true, 0, goal, 0);
      refine(true, 0, goal);
    }
  }

  // The draw.
  u64 rank_of_tie = 0, run_ties = 0;
  const bool from_list = listed && !use_m;
  if (from_list) {
    // What stays of the window, by the thread in whose run it is.
    const float cut_v = cut_key == 0 ? -INFINITY : cut_value(cut_key);
    R.clear(true);
    for_window([&](float v, int i) {
      if (v > cut_v)
        R.add_mass(i / run_len, weight(v));
      else if (v == cut_v)
        atomicAdd(&sh.count[i / run_len], 1u);
    });
    __syncthreads();
    run_ties = sh.count[tid];
    if (cut_ties < cut_all) {
      u64 all;
      rank_of_tie = R.prefix(run_ties, all);
    }
  } else if (cut_ties < cut_all) {
    u64 ties = 0, all;
    const float cut_v = cut_value(cut_key);
    for (int i = i0; i < i1; ++i) ties += elem(i) == cut_v;
    rank_of_tie = R.prefix(ties, all);
  }
  u64 mine = 0, total;
  if (from_list) {
    const u64 left = rank_of_tie < cut_ties ? cut_ties - rank_of_tie : 0;
    mine = run_sum + sh.mass[0][tid] + (static_cast<u64>(sh.mass[1][tid]) << 16) + (static_cast<u64>(sh.mass[2][tid]) << 32);
    if (cut_key != 0) mine += min64(run_ties, left) * weight(cut_value(cut_key));
  } else if (cut_key == 0 && !use_m) {
    over_run([&](float v, int) { mine += weight(v); });
  } else {
    // What is summed already is not evaluated again (min_p may cut in front of the window).
    const bool summed = run_top < INFINITY && !use_m;
    const float cut_v = cut_key == 0 ? -INFINITY : cut_value(cut_key);
    if (summed) mine = run_sum;
    u64 tie = rank_of_tie;
    for (int i = i0; i < i1; ++i) {
      const float v = elem(i);
      if (v < cut_v || (summed && v > run_top)) continue;
      if (v == cut_v && tie++ >= cut_ties) continue;
      const u64 w = weight(v);
      if (enough(w)) mine += w;
    }
  }
  const u64 at = R.prefix(mine, total);
  const u64 goal = min64(static_cast<u64>(u * static_cast<double>(total)), total - 1);
  // The thread whose run holds the goal; its warp walks the run.
  const uint32_t owner = __ballot_sync(0xffffffffu, at <= goal && goal < at + mine);
  if (owner != 0) {
    const int o = __ffs(static_cast<int>(owner)) - 1, lane = tid & 31;
    const int w0 = __shfl_sync(0xffffffffu, i0, o), w1 = __shfl_sync(0xffffffffu, i1, o);
    u64 base = __shfl_sync(0xffffffffu, at, o), tie = __shfl_sync(0xffffffffu, rank_of_tie, o);
    for (int i = w0; i < w1; i += 32) {
      const float v = i + lane < w1 ? elem(i + lane) : -INFINITY;
      const uint32_t key = cut_key_of(v);
      const uint32_t ties = __ballot_sync(0xffffffffu, i + lane < w1 && key == cut_key);
      const bool out = i + lane >= w1 || key < cut_key ||
                       (key == cut_key && tie + __popc(ties & ((1u << lane) - 1)) >= cut_ties);
      u64 w = out ? 0 : weight(v);
      if (!enough(w)) w = 0;
      u64 inc = w;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const u64 nb = __shfl_up_sync(0xffffffffu, inc, s);
        if (lane >= s) inc += nb;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, goal < base + inc);
      if (hit != 0) {
        if (lane == __ffs(static_cast<int>(hit)) - 1) {
          p.token[row] = first + i + lane;
          if (p.logprob) p.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total)));
        }
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
      tie += __popc(ties);
    }
  }
  if (ranks > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <class E, int kThreads, bool kStaged, Filters kFilters>
int launch_typed(SampleArgs p, int64_t B, int64_t c, int dev, cudaStream_t stream) {
  static std::atomic<uint64_t> attr_set{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (!(attr_set.load() & bit)) {
    KW8_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<E, kThreads, kStaged, kFilters>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    KW8_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<E, kThreads, kStaged, kFilters>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_set.fetch_or(bit);
  }
  p.slice = static_cast<int>((p.V + c - 1) / c);
  const size_t smem = sizeof(SampShared) + (kStaged ? static_cast<size_t>(p.slice) * sizeof(E) + 16 : 0);
  KW8_REQUIRE(p.slice <= 65535 && smem <= static_cast<size_t>(kMaxSmem), KW8_ERR_UNSUPPORTED,
              "vocabulary of %d too large", p.V);
  KW8_REQUIRE(B * c < (1ll << 31), KW8_ERR_UNSUPPORTED, "too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B * c), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(c);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  KW8_CUDA_TRY(cudaLaunchKernelEx(&cfg, sample_kernel<E, kThreads, kStaged, kFilters>, p));
  return KW8_OK;
}

// CTAs per row: a power of two up to sixteen (other sizes pack badly into the
// GPCs: 64 rows of 151936 bf16, top-k 50: 4 CTAs 23 us, 5 to 8 35 to 41 us).
// One CTA per SM while every row has the same settings: a second one next to it
// costs more in exchanges than it gains (256 x 32000 bf16: 1 CTA a row 20 us, 2
// 30 us).  With settings of one per row the slowest rows bound the launch, and
// up to four waves of smaller CTAs even them out (64 x 151643 fp32: 4 CTAs a
// row 56 us, 8 51 us, 16 65 us).
template <class E>
int launch_split(const SampleArgs& p, int64_t B, cudaStream_t stream) {
  int dev = 0;
  KW8_CUDA_TRY(cudaGetDevice(&dev));
  const int64_t sms = num_sms(dev);
  const bool per_row = p.temperature || p.top_k || p.top_p || p.min_p;
  const int64_t most = per_row ? 4 * sms : sms;
  int64_t c = per_row ? 8 : 16;
  while (c > 1 && (c * B > most || p.V / c < 2048)) c /= 2;
  constexpr int64_t fit = std::min<int64_t>(
      65535, (kMaxSmem - 16 - static_cast<int64_t>(sizeof(SampShared))) / static_cast<int64_t>(sizeof(E)));
  static_assert(kMaxRanks * fit >= kSampleMaxV, "the largest vocabulary must fit into a cluster's shared memory");
  while (c < kMaxRanks && c * fit < p.V) c *= 2;
  // Slices that leave room for one CTA per SM only, and more CTAs than SMs: read
  // from L1 and L2 again, so that two CTAs share an SM (64 x 151936 fp32 top-k 50:
  // 25 us, staged 36; top-p 0.9: 72 against 86).  Not where every token is
  // weighed and nothing filtered (256 x 32000 fp32: 26 us, staged 24).
  const int64_t smem = static_cast<int64_t>(sizeof(SampShared)) + (p.V + c - 1) / c * static_cast<int64_t>(sizeof(E)) + 16;
  const bool staged = smem <= 113 * 1024 || c * B <= sms;
  if (!p.top_k && p.top_k0 > 0 && p.top_k0 < p.V)
    return staged ? launch_typed<E, 512, true, kTopK>(p, B, c, dev, stream) : launch_typed<E, 512, false, kTopK>(p, B, c, dev, stream);
  if (!p.top_k && !p.top_p && !p.min_p && !(p.top_p0 < 1.f) && !(p.min_p0 > 0.f))
    return launch_typed<E, 512, true, kNone>(p, B, c, dev, stream);
  if (!p.top_k)
    return staged ? launch_typed<E, 512, true, kNoTopK>(p, B, c, dev, stream) : launch_typed<E, 512, false, kNoTopK>(p, B, c, dev, stream);
  return staged ? launch_typed<E, 512, true, kAny>(p, B, c, dev, stream) : launch_typed<E, 512, false, kAny>(p, B, c, dev, stream);
}

}  // namespace

int launch_sample(const SampleArgs& args, int64_t B, int logits_dtype, cudaStream_t stream) {
  return logits_dtype == KW8_DT_F32 ? launch_split<float>(args, B, stream)
                                    : launch_split<__nv_bfloat16>(args, B, stream);
}

}  // namespace kw8
