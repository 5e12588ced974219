// W8A8 linear: kernels and launcher (see gemm_q8.cuh).
#include "gemm_q8.cuh"

#include "gemm_tc.cuh"
#include "pack.cuh"

namespace kw8 {

namespace {

constexpr int kQ8BK = 128;             // k per stage: one 128-byte swizzle row
constexpr int kQ8Rows = 128;           // M of the MMA
constexpr int kQ8MaxStages = 12;
constexpr int kQ8Threads = 256;
constexpr int kQ8ABytes = kQ8Rows * kQ8BK;  // 16 KB

// D[tmem] (+)= A[smem] x B[smem]^T, kind::i8 (int8 operands, int32 sums).
__device__ __forceinline__ void mma_ss_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor, kind::i8: A = B = signed 8 bit (both K-major), D = s32.
__device__ __forceinline__ uint32_t idesc_i8_s32(uint32_t M, uint32_t N) {
  return (2u << 4)            // D format: s32
         | (1u << 7)          // A format: signed
         | (1u << 10)         // B format: signed
         | ((N >> 3) << 17)   // N / 8
         | ((M >> 4) << 24);  // M / 16
}

// Shared-memory matrix descriptor of a K-major operand without swizzle: 8-row
// groups of 16-byte chunks (128 contiguous bytes), chunks 128 B apart along
// k, groups 512 B apart along the rows: the tiled weight layout as it is.
__device__ __forceinline__ uint64_t smem_desc_kmajor_tiled(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 16;  // LBO
  d |= static_cast<uint64_t>(512 >> 4) << 32;  // SBO
  d |= static_cast<uint64_t>(1) << 46;         // descriptor version
  return d;
}

// The weights are the MMA's A operand (M = 128 output channels), the rows of
// q its B operand (N = nt rows).  One tile per CTA of 256 threads:
//   warp 0  TMA producer: a 16 KB weight box and an nt x 128 B row box per stage;
//   warp 1  MMA issuer: four tcgen05.mma (K = 32) per stage, one commit;
//   all     epilogue: warps w and w + 4 read the output channels (TMEM lanes)
//           32 (w mod 4).., alternate 16-row chunks.
// With k_splits > 1 the CTAs of a cluster each take a range of the k tiles and
// add their int32 sums through distributed shared memory: whole numbers, so the
// split changes no bit.  Bound by the weight bytes for few rows.
__global__ void __launch_bounds__(kQ8Threads)
    linear_q8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                     const Q8LinearArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full[kQ8MaxStages], empty[kQ8MaxStages], acc_full;
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int stages = p.stages, nt = p.nt;
  const int stage_bytes = kQ8ABytes + nt * kQ8BK;
  uint32_t cols = 32;
  while (cols < static_cast<uint32_t>(nt)) cols *= 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    abort_sh = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) tmem_alloc(&tmem_base_sh, cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  volatile int* abort_flag = &abort_sh;
  const uint32_t tmem = tmem_base_sh;

  const int ks = p.k_splits;
  const int rank = ks > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  // Tiles of the same weights are neighbours, so that their second and later reads come from L2.
  const int t_tiles = (p.T + nt - 1) / nt;
  const int ft = static_cast<int>(blockIdx.x / ks) / t_tiles;  // feature tile
  const int t0 = (static_cast<int>(blockIdx.x / ks) - ft * t_tiles) * nt;
  const int k_tiles = (p.K + kQ8BK - 1) / kQ8BK;
  const int per = (k_tiles + ks - 1) / ks;
  const int kt0 = min(k_tiles, rank * per), kt1 = min(k_tiles, kt0 + per);

  // Whole warps go through these loops, so that addresses and descriptors stay
  // in uniform registers; one elected lane issues.  (One lane's own loop needs
  // about 100 cycles per MMA.)  Passing a barrier is slow too, so the next
  // stage's is looked at before this stage's work.
  if (warp == 0) {
    const bool elected = elect_one();
    uint32_t phase = 0, armed = 0, armed_phase = 0;  // bit s: stage s was armed, and in which phase last
    int stage = 0;
    bool ready = false;
    for (int kt = kt0; kt < kt1; ++kt) {
      if (!ready && !__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, abort_flag))) break;
      const int next = stage + 1 == stages ? 0 : stage + 1;
      const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
      const bool peek = mbar_test_wait(&empty[next], next_phase ^ 1u);
      armed |= 1u << stage;
      armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
      uint8_t* dst = smem + stage * stage_bytes;
      if (elected) {
        mbar_arrive_expect_tx(&full[stage], stage_bytes);
        if (p.w_tiled) {
          tma_load_3d(dst, &map_w, &full[stage], 0, kt * 8, ft * (kQ8Rows / 16));
          tma_load_3d(dst + kQ8ABytes / 2, &map_w, &full[stage], 0, kt * 8 + 4, ft * (kQ8Rows / 16));
        } else {
          tma_load_2d(dst, &map_w, &full[stage], kt * kQ8BK, ft * kQ8Rows);
        }
        tma_load_2d(dst + kQ8ABytes, &map_x, &full[stage], kt * kQ8BK, t0);
      }
      __syncwarp();
      ready = __all_sync(0xffffffffu, peek);
      stage = next;
      phase = next_phase;
    }
    // No load may still be on its way into this CTA's memory when it goes on
    // (also after a wait that gave up): wait, bounded, for what was armed.
    if (lane == 0)
      for (int s = 0; s < stages; ++s)
        if (armed & (1u << s)) mbar_wait(&full[s], (armed_phase >> s) & 1u, nullptr);
  } else if (warp == 1) {
    const bool elected = elect_one();
    const uint32_t idesc = idesc_i8_s32(kQ8Rows, static_cast<uint32_t>(nt));
    const uint32_t smem0 = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t a_desc0 = p.w_tiled ? smem_desc_kmajor_tiled(smem0) : smem_desc_kmajor_sw128(smem0);
    const uint64_t b_desc0 = smem_desc_kmajor_sw128(smem0 + kQ8ABytes);
    // k step of 32 in the weights' box, in 16-byte units.
    const uint32_t a_k1 = p.w_tiled ? 16 : 2, a_k2 = p.w_tiled ? kQ8ABytes / 32 : 4;
    uint32_t phase = 0;
    int stage = 0;
    bool ready = false;
    for (int kt = kt0; kt < kt1; ++kt) {
      if (!ready && !__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort_flag))) break;
      const int next = stage + 1 == stages ? 0 : stage + 1;
      const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
      const bool peek = mbar_test_wait(&full[next], next_phase);
      tc_fence_after();
      const uint32_t off = static_cast<uint32_t>(stage * stage_bytes) >> 4;
      const uint64_t ad = a_desc0 + off, bd = b_desc0 + off;
      if (elected) {
        mma_ss_i8(tmem_u, ad, bd, idesc, kt != kt0 ? 1u : 0u);
        mma_ss_i8(tmem_u, ad + a_k1, bd + 2, idesc, 1u);
        mma_ss_i8(tmem_u, ad + a_k2, bd + 4, idesc, 1u);
        mma_ss_i8(tmem_u, ad + a_k2 + a_k1, bd + 6, idesc, 1u);
        mma_commit(&empty[stage]);
      }
      __syncwarp();
      ready = __all_sync(0xffffffffu, peek);
      stage = next;
      phase = next_phase;
    }
    if (elected) mma_commit(&acc_full);  // every MMA above has completed once this arrives
  }
  __syncwarp();
  const bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full, 0, nullptr));
  tc_fence_after();
  const int q = warp & 3, half = warp >> 2;
  const int f = ft * kQ8Rows + q * 32 + lane;
  const bool fvalid = f < p.N;
  const float sw = load_scale(p.w_scale, p.w_scale_dtype, p.w_scale_pc && fvalid ? f : 0);
  const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16);
  const int left = min(nt, p.T - t0);
  if (ks == 1) {
    for (int c = half * 16; c < left && ok; c += 32) {
      uint32_t r[16];
      KW8_TMEM_LD_X16(acc + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (fvalid && c + j < left) {
          const float y = static_cast<float>(static_cast<int>(r[j])) * __ldg(p.x_scale + t0 + c + j) * sw;
          const int64_t o = static_cast<int64_t>(t0 + c + j) * p.N + f;
          if (p.out_f32)
            static_cast<float*>(p.out)[o] = y;
          else
            static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(y);
        }
    }
  } else {
    // Partial sums [row][128 channels] over the ring (its loads are consumed).
    int* part = reinterpret_cast<int*>(smem);
    for (int c = half * 16; c < nt; c += 32) {
      uint32_t r[16];
      KW8_TMEM_LD_X16(acc + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j) part[(c + j) * kQ8Rows + q * 32 + lane] = kt0 < kt1 ? static_cast<int>(r[j]) : 0;
    }
    cluster_sync_all();
    // Rows rank, rank + ks, ...: this CTA's share of the tile; a warp per row,
    // four channels per lane.
    const uint32_t base = smem_u32(part) + lane * 16;
    const int f4 = ft * kQ8Rows + lane * 4;
    float sw4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sw4[i] = load_scale(p.w_scale, p.w_scale_dtype, p.w_scale_pc ? min(f4 + i, p.N - 1) : 0);
    const int64_t esize = p.out_f32 ? 4 : 2;
    const bool vec = f4 + 4 <= p.N && p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & (4 * esize - 1)) == 0;
    constexpr int kRows = 4, kWarps = kQ8Threads / 32;  // rows in flight per warp
    for (int i0 = warp; rank + i0 * ks < left && ok; i0 += kWarps * kRows) {
      int4 sum[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) sum[i] = make_int4(0, 0, 0, 0);
      for (int s = 0; s < ks; ++s) {
        const uint32_t at = mapa_shared(base, static_cast<uint32_t>(s));
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int t = rank + (i0 + kWarps * i) * ks;
          if (t < left) {
            int4 v;
            asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(at + static_cast<uint32_t>(t) * (kQ8Rows * 4)));
            sum[i].x += v.x; sum[i].y += v.y; sum[i].z += v.z; sum[i].w += v.w;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int t = rank + (i0 + kWarps * i) * ks;
        if (t >= left || f4 >= p.N) continue;
        const float sx = __ldg(p.x_scale + t0 + t);
        const float y[4] = {static_cast<float>(sum[i].x) * sx * sw4[0], static_cast<float>(sum[i].y) * sx * sw4[1],
                            static_cast<float>(sum[i].z) * sx * sw4[2], static_cast<float>(sum[i].w) * sx * sw4[3]};
        const int64_t o = static_cast<int64_t>(t0 + t) * p.N + f4;
        if (p.out_f32) {
          float* dst = static_cast<float*>(p.out) + o;
          if (vec) {
            *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
          } else {
            for (int j = 0; j < 4; ++j)
              if (f4 + j < p.N) dst[j] = y[j];
          }
        } else {
          __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + o;
          if (vec) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          } else {
            for (int j = 0; j < 4; ++j)
              if (f4 + j < p.N) dst[j] = __float2bfloat16_rn(y[j]);
          }
        }
      }
    }
    cluster_sync_all();  // no CTA leaves while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// ---------------------------------------------------------------- pairs --
//
// Many rows: tiles of 256 rows of q by nt output channels over a CTA pair
// (tcgen05.mma cta_group::2, M = 256).  Each CTA stages its own 128 rows of q
// and half of the tile's weight rows, so a stage of 128 k costs an SM 32 KB of
// L2 and shared-memory traffic for 64 Kmul-adds a byte: with one CTA per tile
// the weights (nt x 128 B) and their second read by the tensor core would take
// longer than the MMAs.  Persistent over tiles, two accumulators in TMEM, so
// the epilogue of one tile runs beside the next one's MMAs.
//   warps 0, 3  TMA producers of the rows of q and of the weights; both CTAs'
//               loads complete on CTA 0's `full`;
//   warp 1      CTA 0: MMA issuer for the pair; commits free the stage in both;
//   warp 2      TMEM allocation;
//   warps 4..11 epilogue of the CTA's 128 rows, two warps per 32 rows
//               (alternate boxes): TMEM -> scales -> a swizzled
//               32-row box in shared memory -> TMA store (word stores, a row at a
//               time, where the output's rows are no 16-byte multiples).

constexpr int kQ8PairEpiWarps = 8;
constexpr int kQ8PairThreads = 128 + 32 * kQ8PairEpiWarps;
constexpr int kQ8PairMaxStages = 8;
constexpr int kQ8BoxBytes = 32 * 128;  // one warp's output box

struct Q8PairArgs {
  Q8LinearArgs g;
  int t_tiles, n_tiles;
  int boxes;  // output boxes per epilogue warp (1 or 2)
};

__device__ __forceinline__ void mma_ss_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// TMA load into this CTA's shared memory that completes on a barrier of either
// CTA of the pair (shared::cluster address).  No multicast.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t smem_dst, const CUtensorMap* map, uint32_t bar_cluster,
                                                 int32_t c0, int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar_cluster)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t smem_dst, const CUtensorMap* map, uint32_t bar_cluster,
                                                 int32_t c0, int32_t c1, int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar_cluster)
      : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* smem_src, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(smem_u32(smem_src))
               : "memory");
}

template <bool kF32, bool kTma>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kQ8PairThreads, 1)
    linear_q8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                          const __grid_constant__ CUtensorMap map_out, const Q8PairArgs pa) {
  const Q8LinearArgs& p = pa.g;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full[kQ8PairMaxStages], empty[kQ8PairMaxStages], acc_full[2], acc_empty[2], drain_bar;
  __shared__ __align__(16) float sw_sh[kQ8PairEpiWarps][256];  // read as float4
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const bool leader = crank == 0;
  const int stages = p.stages, nt = p.nt, half = nt / 2;
  const int stage_bytes = kQ8ABytes + half * kQ8BK;
  uint8_t* const boxes = smem + stages * stage_bytes;  // one or two output boxes per epilogue warp

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kQ8PairEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    abort_sh = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    if (kTma) tma_prefetch_desc(&map_out);
  }
  if (warp == 2) tmem_alloc_pair(&tmem_base_sh, kTcTmemCols);
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers are initialised, TMEM allocated
  tc_fence_after();
  volatile int* abort_flag = &abort_sh;
  const uint32_t tmem = tmem_base_sh;

  const int k_tiles = (p.K + kQ8BK - 1) / kQ8BK;
  const int total = pa.t_tiles * pa.n_tiles;
  const int first = static_cast<int>(blockIdx.x >> 1), step = static_cast<int>(gridDim.x >> 1);

  if (warp == 0 || warp == 3) {
    const bool elected = elect_one();
    const bool rows = warp == 0;  // the rows of q, and CTA 0's arming of the stage; else the weights
    const uint32_t smem0 = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
    const uint32_t full0 = __shfl_sync(0xffffffffu, mapa_shared(smem_u32(&full[0]), 0), 0);  // CTA 0's
    uint32_t phase = 0, armed = 0, armed_phase = 0;
    int stage = 0;
    bool ok = true, ready = false;
    for (int t = first; ok && t < total; t += step) {
      const int t0 = (t % pa.t_tiles) * 256 + static_cast<int>(crank) * kQ8Rows;
      const int n0 = (t / pa.t_tiles) * nt + static_cast<int>(crank) * half;
      for (int kt = 0; kt < k_tiles; ++kt) {
        if (!ready && !__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, abort_flag))) {
          ok = false;
          break;
        }
        const int next = stage + 1 == stages ? 0 : stage + 1;
        const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
        const bool peek = mbar_test_wait(&empty[next], next_phase ^ 1u);
        const uint32_t dst = smem0 + static_cast<uint32_t>(stage * stage_bytes);
        const uint32_t bar = full0 + static_cast<uint32_t>(stage) * 8;
        if (rows) {
          if (elected) {
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * stage_bytes);
            tma_load_2d_pair(dst, &map_x, bar, kt * kQ8BK, t0);
          }
          armed |= 1u << stage;
          armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
        } else if (p.w_tiled) {
          if (elected) {
            tma_load_3d_pair(dst + kQ8ABytes, &map_w, bar, 0, kt * 8, n0 / 16);
            tma_load_3d_pair(dst + kQ8ABytes + half * 64, &map_w, bar, 0, kt * 8 + 4, n0 / 16);
          }
        } else if (elected) {
          tma_load_2d_pair(dst + kQ8ABytes, &map_w, bar, kt * kQ8BK, n0);
        }
        __syncwarp();
        ready = __all_sync(0xffffffffu, peek);
        stage = next;
        phase = next_phase;
      }
    }
    // No load may still be under way when the CTAs leave: CTA 0 waits
    // (bounded) for both CTAs' bytes of what it armed.
    if (leader && rows && lane == 0)
      for (int s = 0; s < stages; ++s)
        if (armed & (1u << s)) mbar_wait_cluster(&full[s], (armed_phase >> s) & 1u, nullptr);
    __syncwarp();
  } else if (warp == 1) {
    if (leader) {
      // The whole warp goes through the loop, so that descriptors stay in
      // uniform registers; one elected lane issues.
      const bool elected = elect_one();
      const uint32_t idesc = idesc_i8_s32(256, static_cast<uint32_t>(nt));
      const uint32_t smem0 = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t a_desc0 = smem_desc_kmajor_sw128(smem0);
      const uint64_t b_desc0 = p.w_tiled ? smem_desc_kmajor_tiled(smem0 + kQ8ABytes) : smem_desc_kmajor_sw128(smem0 + kQ8ABytes);
      // k step of 32 in the weights' box, in 16-byte units.
      const uint32_t b_k1 = p.w_tiled ? 16 : 2, b_k2 = p.w_tiled ? half * 4 : 4;
      uint32_t phase = 0, acc_phase = 0;
      int stage = 0, done = 0;
      bool ok = true, ready = false;
      for (int t = first; ok && t < total; t += step, ++done) {
        const int ab = done & 1;
        if (!__all_sync(0xffffffffu, mbar_wait_cluster(&acc_empty[ab], ((acc_phase >> ab) & 1u) ^ 1u, abort_flag))) break;
        tc_fence_after();
        const uint32_t d = tmem_u + static_cast<uint32_t>(ab * 256);
        for (int kt = 0; kt < k_tiles; ++kt) {
          // Passing a barrier costs this warp more than an MMA, so the next
          // stage's is looked at before this stage's MMAs are issued.
          if (!ready && !__all_sync(0xffffffffu, mbar_wait_cluster(&full[stage], phase, abort_flag))) {
            ok = false;
            break;
          }
          const int next = stage + 1 == stages ? 0 : stage + 1;
          const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
          const bool peek = mbar_test_wait_cluster(&full[next], next_phase);
          tc_fence_after();
          const uint32_t off = static_cast<uint32_t>(stage * stage_bytes) >> 4;
          const uint64_t ad = a_desc0 + off, bd = b_desc0 + off;
          if (elected) {
            mma_ss_i8_pair(d, ad, bd, idesc, kt != 0 ? 1u : 0u);
            mma_ss_i8_pair(d, ad + 2, bd + b_k1, idesc, 1u);
            mma_ss_i8_pair(d, ad + 4, bd + b_k2, idesc, 1u);
            mma_ss_i8_pair(d, ad + 6, bd + b_k2 + b_k1, idesc, 1u);
            mma_commit_pair(&empty[stage]);
          }
          __syncwarp();
          ready = __all_sync(0xffffffffu, peek);
          stage = next;
          phase = next_phase;
        }
        if (!ok) break;
        if (elected) mma_commit_pair(&acc_full[ab]);
        __syncwarp();
        acc_phase ^= 1u << ab;
      }
      if (elected) mma_commit_pair(&drain_bar);  // arrives in both CTAs once every MMA above has completed
      __syncwarp();
      if (lane == 0) mbar_wait(&drain_bar, 0, nullptr);  // nothing reads or writes this CTA's memory any more
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int q = warp & 3;
    const int half_of = (warp - 4) >> 2;  // which of the boxes: half_of, half_of + 2, ...
    float* const sw = sw_sh[warp - 4];
    uint8_t* const my_boxes = boxes + (warp - 4) * pa.boxes * kQ8BoxBytes;
    const uint32_t acc_lane = tmem + (static_cast<uint32_t>(q * 32) << 16);
    constexpr int kCols = kF32 ? 32 : 64;  // of a box: 128 bytes
    const auto first_row = [&](int t) { return (t % pa.t_tiles) * 256 + static_cast<int>(crank) * kQ8Rows + q * 32; };
    // The scales of the next tile are fetched while this one is stored.
    float next_sx = 0.f, next_sw[8];
    const auto fetch = [&](int t) {
      const int r = first_row(t) + lane, n0 = (t / pa.t_tiles) * nt;
      next_sx = r < p.T ? __ldg(p.x_scale + r) : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = i * 32 + lane;
        next_sw[i] = c < nt && n0 + c < p.N ? load_scale(p.w_scale, p.w_scale_dtype, p.w_scale_pc ? n0 + c : 0) : 0.f;
      }
    };
    if (first < total) fetch(first);
    uint32_t acc_phase = 0;
    int done = 0, used = 0;
    for (int t = first; t < total; t += step, ++done) {
      const int ab = done & 1;
      const int r0 = first_row(t), n0 = (t / pa.t_tiles) * nt;
      const float sx = next_sx;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) sw[i * 32 + lane] = next_sw[i];
      __syncwarp();
      if (t + step < total) fetch(t + step);
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[ab], (acc_phase >> ab) & 1u, abort_flag))) break;
      tc_fence_after();
      const uint32_t acc = acc_lane + static_cast<uint32_t>(ab * 256);
      const bool rows_here = r0 < p.T;
      for (int c0 = half_of * kCols; c0 < nt && rows_here && n0 + c0 < p.N; c0 += 2 * kCols, ++used) {
        uint32_t r[kCols];
        KW8_TMEM_LD_X32(acc + c0, r);
        if constexpr (!kF32) {
          uint32_t* const r2 = r + 32;
          KW8_TMEM_LD_X32(acc + c0 + 32, r2);
        }
        uint8_t* const b = my_boxes + (used & (pa.boxes - 1)) * kQ8BoxBytes;
        if constexpr (kTma) {
          // The box's last store has been read.
          if (lane == 0) {
            if (pa.boxes == 2)
              asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            else
              asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          }
          __syncwarp();
        }
        tmem_wait_ld();
        const float4* s4 = reinterpret_cast<const float4*>(sw + c0);
        const int left = p.N - (n0 + c0);
        // Row `lane` of the box: 32 words, 16-byte chunk c at c ^ (lane & 7) (the 128-byte swizzle).
        uint8_t* const row = b + lane * 128;
        const uintptr_t row_out = reinterpret_cast<uintptr_t>(p.out) +
                                  (static_cast<uintptr_t>(r0 + lane) * static_cast<uintptr_t>(p.N) + n0 + c0) * (kF32 ? 4 : 2);
        const bool odd = !kF32 && !kTma && (row_out & 2) != 0;
        uint32_t carry = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t o[4];
          if constexpr (kF32) {
            const float4 s = s4[c];
            o[0] = __float_as_uint(static_cast<float>(static_cast<int>(r[4 * c])) * sx * s.x);
            o[1] = __float_as_uint(static_cast<float>(static_cast<int>(r[4 * c + 1])) * sx * s.y);
            o[2] = __float_as_uint(static_cast<float>(static_cast<int>(r[4 * c + 2])) * sx * s.z);
            o[3] = __float_as_uint(static_cast<float>(static_cast<int>(r[4 * c + 3])) * sx * s.w);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float4 s = s4[2 * c + i];
              const int j = 8 * c + 4 * i;
              const __nv_bfloat162 lo = __floats2bfloat162_rn(static_cast<float>(static_cast<int>(r[j])) * sx * s.x,
                                                              static_cast<float>(static_cast<int>(r[j + 1])) * sx * s.y);
              const __nv_bfloat162 hi = __floats2bfloat162_rn(static_cast<float>(static_cast<int>(r[j + 2])) * sx * s.z,
                                                              static_cast<float>(static_cast<int>(r[j + 3])) * sx * s.w);
              o[2 * i] = *reinterpret_cast<const uint32_t*>(&lo);
              o[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hi);
            }
            if constexpr (!kTma) {
              // A row whose output starts inside a word: the box holds the
              // output's words, one value later.
              if (odd) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t w = __byte_perm(carry, o[i], 0x5432);
                  carry = o[i];
                  o[i] = w;
                }
              }
            }
          }
          *reinterpret_cast<uint4*>(row + ((c ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        if constexpr (kTma) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_out, b, n0 + c0, r0);  // rows and channels past the end are not written
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          // Output rows that are no 16-byte multiples: a row of the box at a time, one word per lane.
          __syncwarp();
          const int rows = min(32, p.T - r0);
          // The row's first word (its values may start in the word's upper half: o = 1) and the step to the next row's.
          const uintptr_t start = reinterpret_cast<uintptr_t>(p.out) +
                                  (static_cast<uintptr_t>(r0) * static_cast<uintptr_t>(p.N) + n0 + c0) * (kF32 ? 4 : 2);
          uint32_t* dst = reinterpret_cast<uint32_t*>(start & ~static_cast<uintptr_t>(3)) + lane;
          int o = kF32 ? 0 : static_cast<int>((start >> 1) & 1);
          const int words = kF32 ? p.N : p.N >> 1, half_word = kF32 ? 0 : p.N & 1;
          // Whole words only: word `lane` holds values 2 lane - o and the next.
          const bool whole[2] = {kF32 ? lane < left : 2 * lane + 1 < left, !kF32 && lane > 0 && 2 * lane < left};
          constexpr int kAtOnce = 8;
          for (int i0 = 0; i0 < rows; i0 += kAtOnce) {
            uint32_t v[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
              v[i] = *reinterpret_cast<const uint32_t*>(b + (i0 + i) * 128 + (((lane >> 2) ^ ((i0 + i) & 7)) << 4) + (lane & 3) * 4);
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
              if (i0 + i < rows && (o ? whole[1] : whole[0])) *dst = v[i];
              dst += words + (o & half_word);
              o ^= half_word;
            }
          }
          if constexpr (!kF32) {
            // The values at the ends that share their word with another row or box.
            if (lane < rows) {
              uint16_t* const dst = reinterpret_cast<uint16_t*>(row_out);
              const int last = min(left, 64) - 1;
              const auto at = [&](int k) -> uint16_t {  // half k of the row's words
                return static_cast<uint16_t>(
                    *reinterpret_cast<const uint32_t*>(row + (((k >> 3) ^ (lane & 7)) << 4) + ((k >> 1) & 3) * 4) >> (16 * (k & 1)));
              };
              if (odd) {
                dst[0] = at(1);
                if (last == 63) dst[63] = static_cast<uint16_t>(carry >> 16);
                else if (last > 0 && (last & 1)) dst[last] = at(last + 1);
              } else if ((last & 1) == 0) {
                dst[last] = at(last);
              }
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[ab]), 0));
      acc_phase ^= 1u << ab;
    }
    if (kTma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    // CTA 1 waits for the MMAs here, behind its tiles: from the start, the wait's
    // limit would cover the whole launch (180224 x 131056 x 180224 takes more) and
    // report a timeout where everything goes on.
    if (!leader && warp == 4 && lane == 0) mbar_wait(&drain_bar, 0, nullptr);
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base_sh, kTcTmemCols);
  }
}

// TMEM columns of a tile of nt columns.
int q8_cols(int nt) {
  int c = 32;
  while (c < nt) c *= 2;
  return c;
}

// The choice between the two kernels, their tiles and the K splits is the least
// of these models (us beyond a common part), fitted to 657 shapes of 17 to 1000
// rows, K 64 to 9728 and 64 to 40960 channels: 1.9% above the best of the
// measured choices on average, more than 10% at 49 of them, 31% at worst (33 to 64
// rows of 9728 x 20480: 32-row tiles 51 us, the best 39 to 40).  Outside of that,
// measured afterwards: heads of 151936 channels, 1 to 300 rows, K 1024 to 2560: always
// the best; 1500 to 8192 rows, K 64 to 4096, 64 to 8192 channels: 1.2% above it on
// average, 25% at worst (8192 x 64 x 64: 6.3 us, pairs 5.0).  Both sides of it: 96 x 2048 x 4096
// 8.4 us here, 7.3 with pairs; 77 x 2560 x 10243 11 us, 12.7 with pairs; 256 x 9728
// x 64 8 us, 15 with pairs; 64 x 2048 x 151936 66 us with 64-row tiles, 74 with
// 32-row ones, 69 with pairs.
//
// One CTA per tile of nt rows: a k tile takes 0.25 us and a tile 1.25 us more
// (2.4 with 64 rows), shared by the CTAs of an SM; the weights come no faster
// than 6 TB/s; joining ks parts of K costs 0.9 + 0.1 ks, and pays only while all
// of them are resident (80 x 2048 x 151936 in 8 parts: 536 us, in one 74).
double plan_single(Q8LinearArgs& p, int dev, int rows) {
  const int64_t T = p.T, N = p.N, K = p.K, k_tiles = (K + kQ8BK - 1) / kQ8BK;
  p.nt = static_cast<int>(std::min<int64_t>(rows, (T + 15) / 16 * 16));
  const double tiles = static_cast<double>((N + kQ8Rows - 1) / kQ8Rows * ((T + p.nt - 1) / p.nt));
  const double sms = num_sms(dev), weights = static_cast<double>(N) * static_cast<double>(K) / 6e6;
  double best = 1e30, total = 0.0;
  for (int ks = 1; ks <= 8; ++ks) {
    if (valid_k_splits(ks, k_tiles) != ks || (ks > 1 && tiles * ks > 2 * sms)) continue;
    const double k_us = static_cast<double>((k_tiles + ks - 1) / ks) * 0.25, tile_us = p.nt <= 32 ? 1.25 : 2.4;
    const double load = std::max(1.0, 0.7 * tiles * ks / sms), join = ks > 1 ? 0.9 + 0.1 * ks : 0.0;
    // The split that does the k tiles fastest (1 x 2048 x 4096: 4 parts 6.0 us, 6 parts 7.5, one 8).
    const double us = std::max(weights, k_us * load) + join;
    if (us < best) {
      best = us;
      p.k_splits = ks;
      total = std::max(weights, (k_us + tile_us) * load) + join;
    }
  }
  return total;
}

// Output rows that a TMA store can write.
bool tma_rows(const Q8LinearArgs& p) {
  return static_cast<int64_t>(p.N) * (p.out_f32 ? 4 : 2) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
}

// Pairs: the channels per tile with the fewest waves, a wave costing its
// channels plus a fixed part; a k tile takes 0.13 us at least, 0.29 at 256
// channels; output rows that TMA cannot store 1.5 us more.
double plan_pair(Q8LinearArgs& p, int dev) {
  const int64_t T = p.T, N = p.N, K = p.K, pairs = num_sms(dev) / 2;
  int64_t best = INT64_MAX, waves = 1;
  for (int nt = 256; nt >= 64; nt -= 64) {
    const int64_t w = ((T + 255) / 256 * ((N + nt - 1) / nt) + pairs - 1) / pairs;
    if (w * (nt + 32) < best) {
      best = w * (nt + 32);
      waves = w;
      p.nt = nt;
    }
  }
  const double k_tile = std::max(0.13, 0.29 * p.nt / 256);
  return std::max(static_cast<double>(N) * static_cast<double>(K) / 6e6,
                  static_cast<double>(waves) * (static_cast<double>((K + kQ8BK - 1) / kQ8BK) * k_tile + 1.0)) +
         (tma_rows(p) ? 1.0 : 2.5);
}

int make_w_map(CUtensorMap* map, const kw8_weight& w, int64_t N, int64_t K, int rows) {
  if (w.layout == KW8_LAYOUT_TILED)
    return make_tmap_tiled(map, w.q, static_cast<uint64_t>(tiled_ftiles(N)), static_cast<uint64_t>(tiled_steps(K)),
                           static_cast<uint32_t>(rows / 16), 1);
  return make_tmap_2d(map, w.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, N, K, K, kQ8BK, rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

int make_x_map(CUtensorMap* map, const int8_t* q, int64_t T, int64_t K, int rows) {
  return make_tmap_2d(map, q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, T, K, K, kQ8BK, rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Once per device and kernel: allow the largest dynamic shared memory.
template <class K>
int allow_smem(K kernel, int dev, std::atomic<uint64_t>& set, int bytes) {
  const uint64_t bit = 1ull << (dev & 63);
  if (!(set.load() & bit)) {
    KW8_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    set.fetch_or(bit);
  }
  return KW8_OK;
}

constexpr int kQ8PairSmem = 232448 - 9216;  // opt-in limit minus the static part

int launch_pair(const int8_t* q, const kw8_weight& w, Q8LinearArgs p, int dev, cudaStream_t stream) {
  const int64_t esize = p.out_f32 ? 4 : 2;
  const bool tma = tma_rows(p);
  const int kind = (p.out_f32 ? 2 : 0) + (tma ? 1 : 0);
  using Kernel = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const Q8PairArgs);
  static const Kernel kernels[4] = {linear_q8_pair_kernel<false, false>, linear_q8_pair_kernel<false, true>,
                                    linear_q8_pair_kernel<true, false>, linear_q8_pair_kernel<true, true>};
  static std::atomic<uint64_t> attr_set[4];
  int rc = allow_smem(kernels[kind], dev, attr_set[kind], kQ8PairSmem);
  if (rc) return rc;
  const int64_t T = p.T, N = p.N, K = p.K, pairs = num_sms(dev) / 2;
  Q8PairArgs a{};
  a.t_tiles = static_cast<int>((T + 255) / 256);
  a.n_tiles = static_cast<int>((N + p.nt - 1) / p.nt);
  const int stage_bytes = kQ8ABytes + p.nt / 2 * kQ8BK;
  // A short K leaves the epilogue little time to hide in: two boxes per warp; a
  // long one is better served by a deeper ring (8192 x 2560 x 10240: two boxes
  // and four stages 148 us, one and five 140; 8192 x 64 x 10240: 56 against 92).
  a.boxes = (K + kQ8BK - 1) / kQ8BK <= 16 ? 2 : 1;
  const int box_bytes = a.boxes * kQ8PairEpiWarps * kQ8BoxBytes;
  p.stages = std::min(kQ8PairMaxStages, (kQ8PairSmem - 1024 - box_bytes) / stage_bytes);
  CUtensorMap map_x, map_w, map_out;
  rc = make_x_map(&map_x, q, T, K, kQ8Rows);
  if (!rc) rc = make_w_map(&map_w, w, N, K, p.nt / 2);
  map_out = map_x;
  if (!rc && tma)
    rc = make_tmap_2d(&map_out, p.out, p.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                      static_cast<int>(esize), T, N, N * esize, p.out_f32 ? 32 : 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  a.g = p;
  const int64_t grid = 2 * std::min<int64_t>(pairs, static_cast<int64_t>(a.t_tiles) * a.n_tiles);
  kernels[kind]<<<static_cast<unsigned>(grid), kQ8PairThreads, p.stages * stage_bytes + box_bytes + 1024, stream>>>(
      map_x, map_w, map_out, a);
  KW8_CHECK_LAUNCH();
  return KW8_OK;
}

int launch_single(const int8_t* q, const kw8_weight& w, Q8LinearArgs p, int dev, cudaStream_t stream) {
  static std::atomic<uint64_t> attr_set{0};
  int rc = allow_smem(linear_q8_kernel, dev, attr_set, kTcDynSmemMax);
  if (rc) return rc;
  const int64_t T = p.T, N = p.N, K = p.K;
  const int64_t m_tiles = (N + kQ8Rows - 1) / kQ8Rows, t_tiles = (T + p.nt - 1) / p.nt;
  const int stage_bytes = kQ8ABytes + p.nt * kQ8BK;
  // Ring: about 108 KB, two CTAs on an SM (16 x 2560 x 10240: three CTAs of 72
  // KB 10.1 us, two 9.4 us); 72 KB where CTAs follow one another and a third one
  // covers their starts and ends (16 x 2048 x 151936: 56 against 59 us).  Never
  // more CTAs on an SM than its 512 TMEM columns serve, so no allocation waits
  // for another CTA.
  p.stages = std::min(kQ8MaxStages, (m_tiles >= 4 * num_sms(dev) ? 72 : 108) * 1024 / stage_bytes);
  const int smem_bytes = p.stages * stage_bytes + 1024;
  KW8_REQUIRE(p.stages >= 3 && smem_bytes >= q8_cols(p.nt) * 455 &&
                  p.nt * kQ8Rows * 4 <= p.stages * stage_bytes && smem_bytes <= kTcDynSmemMax,
              KW8_ERR_UNSUPPORTED, "no pipeline plan for %d-row tiles", p.nt);
  CUtensorMap map_w, map_x;
  rc = make_w_map(&map_w, w, N, K, kQ8Rows);
  if (!rc) rc = make_x_map(&map_x, q, T, K, p.nt);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(m_tiles * t_tiles * p.k_splits), 1, 1);
  cfg.blockDim = dim3(kQ8Threads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.k_splits);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.k_splits > 1 ? 1 : 0;
  KW8_CUDA_TRY(cudaLaunchKernelEx(&cfg, linear_q8_kernel, map_w, map_x, p));
  return KW8_OK;
}

}  // namespace

int launch_linear_q8(const int8_t* q, const kw8_weight& w, const Q8LinearArgs& args_in, cudaStream_t stream) {
  Q8LinearArgs p = args_in;
  p.w_tiled = w.layout == KW8_LAYOUT_TILED;
  p.w_scale = w.scale;
  p.w_scale_dtype = w.scale_dtype;
  p.w_scale_pc = w.per_channel;
  int dev = 0;
  KW8_CUDA_TRY(cudaGetDevice(&dev));
  Q8LinearArgs narrow = p, wide = p, pair = p;
  const double narrow_us = plan_single(narrow, dev, 32), wide_us = p.T > 32 ? plan_single(wide, dev, 64) : 1e30;
  const double pair_us = p.T > 32 ? plan_pair(pair, dev) : 1e30, single_us = std::min(narrow_us, wide_us);
  if (pair_us < single_us) return launch_pair(q, w, pair, dev, stream);
  return launch_single(q, w, wide_us < narrow_us ? wide : narrow, dev, stream);
}

}  // namespace kw8
