// W8A8 linear: kernels and launcher (see gemm_q8.cuh).
#include "gemm_q8.cuh"

#include "gemm_tc.cuh"
#include "pack.cuh"

namespace kw8 {

namespace {

constexpr int kQ8BK = 128;             // k per stage: one 128-byte swizzle row
constexpr int kQ8Rows = 128;           // M of the MMA
constexpr int kQ8MaxStages = 12;
constexpr int kQ8Threads = 128;
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
// q its B operand (N = nt rows).  One tile per CTA of 128 threads:
//   warp 0  TMA producer: a 16 KB weight box and an nt x 128 B row box per stage;
//   warp 1  MMA issuer: four tcgen05.mma (K = 32) per stage, one commit;
//   all     epilogue: thread i owns output channel i (TMEM lane i).
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  const int ft = blockIdx.x / ks;  // feature tile
  const int t0 = blockIdx.y * nt;
  const int k_tiles = (p.K + kQ8BK - 1) / kQ8BK;
  const int per = (k_tiles + ks - 1) / ks;
  const int kt0 = min(k_tiles, rank * per), kt1 = min(k_tiles, kt0 + per);

  if (warp == 0) {
    if (lane == 0) {
      uint32_t phase = 0, armed = 0, armed_phase = 0;  // bit s: stage s was armed, and in which phase last
      int stage = 0;
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) break;
        armed |= 1u << stage;
        armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
        uint8_t* dst = smem + stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], stage_bytes);
        if (p.w_tiled) {
          tma_load_3d(dst, &map_w, &full[stage], 0, kt * 8, ft * (kQ8Rows / 16));
          tma_load_3d(dst + kQ8ABytes / 2, &map_w, &full[stage], 0, kt * 8 + 4, ft * (kQ8Rows / 16));
        } else {
          tma_load_2d(dst, &map_w, &full[stage], kt * kQ8BK, ft * kQ8Rows);
        }
        tma_load_2d(dst + kQ8ABytes, &map_x, &full[stage], kt * kQ8BK, t0);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // No load may still be on its way into this CTA's memory when it goes on
      // (also after a wait that gave up): wait, bounded, for what was armed.
      for (int s = 0; s < stages; ++s)
        if (armed & (1u << s)) mbar_wait(&full[s], (armed_phase >> s) & 1u, nullptr);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_i8_s32(kQ8Rows, static_cast<uint32_t>(nt));
      uint32_t phase = 0;
      int stage = 0;
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!mbar_wait(&full[stage], phase, abort_flag)) break;
        tc_fence_after();
        const uint32_t a = smem_u32(smem + stage * stage_bytes), b = a + kQ8ABytes;
#pragma unroll
        for (int kk = 0; kk < kQ8BK / 32; ++kk) {
          const uint64_t ad = p.w_tiled ? smem_desc_kmajor_tiled(a + (kk >> 1) * (kQ8ABytes / 2) + (kk & 1) * 256)
                                        : smem_desc_kmajor_sw128(a + kk * 32);
          mma_ss_i8(tmem, ad, smem_desc_kmajor_sw128(b + kk * 32), idesc, (kt != kt0 || kk != 0) ? 1u : 0u);
        }
        mma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      mma_commit(&acc_full);  // every MMA above has completed once this arrives
    }
  }
  __syncwarp();
  const bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full, 0, nullptr));
  tc_fence_after();
  const int f = ft * kQ8Rows + warp * 32 + lane;
  const bool fvalid = f < p.N;
  const float sw = load_scale(p.w_scale, p.w_scale_dtype, p.w_scale_pc && fvalid ? f : 0);
  const uint32_t acc = tmem + (static_cast<uint32_t>(warp * 32) << 16);
  const int left = min(nt, p.T - t0);
  if (ks == 1) {
    for (int c = 0; c < left && ok; c += 16) {
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
    for (int c = 0; c < nt; c += 16) {
      uint32_t r[16];
      KW8_TMEM_LD_X16(acc + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j) part[(c + j) * kQ8Rows + threadIdx.x] = kt0 < kt1 ? static_cast<int>(r[j]) : 0;
    }
    cluster_sync_all();
    const uint32_t base = smem_u32(part);
    // Rows rank, rank + ks, ...: this CTA's share of the tile.
    for (int t = rank; t < left && ok; t += ks) {
      int sum = 0;
      for (int s = 0; s < ks; ++s) {
        int v;
        asm volatile("ld.shared::cluster.s32 %0, [%1];"
                     : "=r"(v)
                     : "r"(mapa_shared(base + (t * kQ8Rows + threadIdx.x) * 4, static_cast<uint32_t>(s))));
        sum += v;
      }
      if (fvalid) {
        const float y = static_cast<float>(sum) * __ldg(p.x_scale + t0 + t) * sw;
        const int64_t o = static_cast<int64_t>(t0 + t) * p.N + f;
        if (p.out_f32)
          static_cast<float*>(p.out)[o] = y;
        else
          static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(y);
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

// TMEM columns of a tile of nt columns.
int q8_cols(int nt) {
  int c = 32;
  while (c < nt) c *= 2;
  return c;
}

}  // namespace

int launch_linear_q8(const int8_t* q, const kw8_weight& w, const Q8LinearArgs& args_in, cudaStream_t stream) {
  Q8LinearArgs p = args_in;
  const int64_t T = p.T, N = p.N, K = p.K;
  p.w_tiled = w.layout == KW8_LAYOUT_TILED;
  p.w_scale = w.scale;
  p.w_scale_dtype = w.scale_dtype;
  p.w_scale_pc = w.per_channel;
  p.nt = static_cast<int>(std::min<int64_t>(128, (T + 15) / 16 * 16));
  const int stage_bytes = kQ8ABytes + p.nt * kQ8BK;
  // Ring: about 72 KB (three CTAs share an SM); never more CTAs on an SM than
  // its 512 TMEM columns serve, so no allocation waits for another CTA.
  p.stages = std::max(3, 73728 / stage_bytes);
  const int smem_bytes = p.stages * stage_bytes + 1024;
  KW8_REQUIRE(p.stages <= kQ8MaxStages && smem_bytes >= q8_cols(p.nt) * 455 && p.nt * kQ8Rows * 4 <= p.stages * stage_bytes &&
                  smem_bytes <= kTcDynSmemMax,
              KW8_ERR_UNSUPPORTED, "no pipeline plan for %d-row tiles", p.nt);
  const int64_t m_tiles = (N + kQ8Rows - 1) / kQ8Rows, t_tiles = (T + p.nt - 1) / p.nt;
  KW8_REQUIRE(t_tiles <= 65535, KW8_ERR_UNSUPPORTED, "too many rows");
  int dev = 0;
  KW8_CUDA_TRY(cudaGetDevice(&dev));
  const int64_t k_tiles = (K + kQ8BK - 1) / kQ8BK;
  const int64_t want = std::min<int64_t>({8, 2 * num_sms(dev) / std::max<int64_t>(1, m_tiles * t_tiles), k_tiles / 2});
  p.k_splits = valid_k_splits(static_cast<int>(std::max<int64_t>(1, want)), k_tiles);

  CUtensorMap map_w, map_x;
  int rc;
  if (p.w_tiled)
    rc = make_tmap_tiled(&map_w, w.q, static_cast<uint64_t>(tiled_ftiles(N)), static_cast<uint64_t>(tiled_steps(K)),
                         kQ8Rows / 16, 1);
  else
    rc = make_tmap_2d(&map_w, w.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, N, K, K, kQ8BK, kQ8Rows,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc)
    rc = make_tmap_2d(&map_x, q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, T, K, K, kQ8BK, p.nt, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  static std::atomic<uint64_t> attr_set{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (!(attr_set.load() & bit)) {
    KW8_CUDA_TRY(cudaFuncSetAttribute(linear_q8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcDynSmemMax));
    attr_set.fetch_or(bit);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(m_tiles * p.k_splits), static_cast<unsigned>(t_tiles), 1);
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

}  // namespace kw8
