// Block-scaled 4-bit GEMM: out = (sum_k a s_a * w s_w) * (s_row x s_col) (+ bias), E2M1 codes with E8M0 (mx) or E4M3 (nv)
// block scales applied by the tensor cores, fp32 accumulation in tensor memory (formats: fp4_common.cuh).
//
// The kernel of small and narrow products (the others run on CTA pairs, gemm_fp4_pair.cu).  One 128 x 64 tile per CTA, 192
// threads: warp 0 fills a ring of {activations, weights, scales of both} stages by TMA, warp 1 copies a stage's scales to
// tensor memory (tcgen05.cp) and issues its four MMAs, warps 2-5 scale, add the bias and store.  Every stage has scale
// columns of its own, so a full stage also says that the MMAs that read them last have completed (its operands could not
// have been overwritten otherwise).
// What bounds it is latency: 3.6 us for a launch of one stage, 0.31 us for every further one (nv; mx 0.25), whatever the
// tile's width.  With few tiles and a long K a cluster of up to eight CTAs splits K: each leaves its fp32 partial tile in
// shared memory, and every CTA adds up and stores a share of the outputs (in rank order, so results do not depend on
// timing).  1 x 5120 -> 1280: 9.9 us by 20 CTAs, 6.2 by 80; 1 x 10240 -> 640: 15.7 by 10, 6.5 by 80.
// Seven stages and one CTA per SM; three stages and two CTAs per SM when there are more tiles than SMs (1 x 1280 -> 10240,
// 160 tiles: 5.5 instead of 9.6 us).  Every wait is bounded; no multicast.
#include "gemm_fp4_common.cuh"

namespace pq {
namespace {

constexpr int BN = 64;                           // tile columns
constexpr int kFp4Threads = 192;
constexpr int kEpiThreads = 128;

template <int FMT, int STAGES>
struct Fp4Smem {
  static constexpr int kABytes = BM * BK;
  static constexpr int kBBytes = BN * BK;
  static constexpr int kOperand = kABytes + kBBytes;
  static constexpr int kScale = Fp4Fmt<FMT>::kScaleBytes;            // per operand
  static constexpr int kScaleOff = STAGES * kOperand;
  static constexpr int kColOff = kScaleOff + STAGES * 2 * kScale;    // s_col, bias: fp32 [BN] each
  static constexpr int kBarOff = kColOff + 2 * BN * 4;
  static constexpr int kMiscOff = kBarOff + (2 * STAGES + 1) * 8;
  static constexpr int kTotal = kMiscOff + 16;
  // What lies over the operand stages once they are used up: the fp32 partial tile of a split launch, or the rounded rows of the
  // output, at a stride of 144 bytes so that eight lanes' 16-byte stores meet different banks.  From there whole rows go out; a lane
  // that stores its own row's pieces took (us, it / this) 560 x 1440 -> 1068 13.5 / 8.5, 1375 x 64 -> 358 12.1 / 7.0, 1024 x 1280 ->
  // 1280 5.9 / 5.7.
  static constexpr int kRedStride = BN + 4;
  static constexpr int kRowStride = 2 * BN + 16;
  static_assert(BM * kRedStride * 4 <= kScaleOff && BM * kRowStride <= kScaleOff, "tiles over the operand stages");
  static_assert(kTotal <= 232448, "exceeds the 227 KB shared memory of one CTA");
  // accumulator, then a set of scale columns per stage
  static constexpr int kSetCols = 2 * 4 * Fp4Fmt<FMT>::kTilesPerStage;
  static constexpr int kCols = BN + STAGES * kSetCols;
  static constexpr int kTmemCols = kCols <= 128 ? 128 : (kCols <= 256 ? 256 : 512);
  static_assert(kCols <= (STAGES == 3 ? 256 : 512), "tensor memory: two CTAs an SM with three stages");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// eight consecutive outputs of one row, columns [col, col + 8)
__device__ __forceinline__ void store8(const Fp4GemmParams& p, int row, int col, const float (&y)[8]) {
  unsigned short* o = static_cast<unsigned short*>(p.out) + static_cast<int64_t>(row) * p.ldo + col;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2_any(y[2 * i], y[2 * i + 1], p.bf16);
  if (p.vec && col + 8 <= p.N) {
    st_v4(o, make_uint4(w[0], w[1], w[2], w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < p.N) o[i] = static_cast<unsigned short>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu);
  }
}
// Up to 64 columns of one output row by a warp, rows that start on any 2-byte border: one 4-byte store per lane from the first
// 4-byte border on, single elements at the ends; n may be zero or less, then nothing is stored.  `read(c)` gives element c.
template <typename Read>
__device__ __forceinline__ void store_row64(unsigned short* o, int n, int lane, Read&& read) {
  const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(o) >> 1) & 1;
  if (n > 64) n = 64;
  const int c = 2 * lane + odd;
  if (odd && lane == 0 && n > 0) o[0] = static_cast<unsigned short>(read(0));
  if (c + 1 < n) *reinterpret_cast<uint32_t*>(o + c) = read(c) | (read(c + 1) << 16);
  else if (c < n) o[c] = static_cast<unsigned short>(read(c));
}

template <int FMT, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(kFp4Threads, STAGES == 3 ? 2 : 1)
pq_fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ CUtensorMap tmT, const __grid_constant__ CUtensorMap tmLb, const Fp4GemmParams p, int split) {
  using L = Fp4Smem<FMT, STAGES>;
  using F = Fp4Fmt<FMT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* done_bar = empty_bar + STAGES;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  float* col_scale = reinterpret_cast<float*>(smem + L::kColOff);
  float* col_bias = col_scale + BN;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = SPLIT ? static_cast<int>(cluster_cta_rank()) : 0;
  const int tile = SPLIT ? static_cast<int>(blockIdx.x) / split : static_cast<int>(blockIdx.x);
  const int row0 = tile % p.mt * BM, n0 = tile / p.mt * BN;
  const int num_kb = (p.K + kFp4StageK - 1) / kFp4StageK;
  const int kb0 = SPLIT ? static_cast<int>(static_cast<int64_t>(num_kb) * rank / split) : 0;
  const int kb1 = SPLIT ? static_cast<int>(static_cast<int64_t>(num_kb) * (rank + 1) / split) : num_kb;
  // the low-rank term is a stage in front of the first CTA's
  const int first = kb0 - (p.t != nullptr && rank == 0 ? 1 : 0);
  const bool aligned_ok = (smem_u32(smem) & 1023u) == 0;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmW);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(done_bar, 1);
    *abort_flag = aligned_ok ? 0 : 1;
    if (!aligned_ok) report_timeout(p.status, 7, 7);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) { tmem_alloc(tmem_holder, L::kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  wait_for_previous_kernel();
  allow_next_kernel();

  if (aligned_ok && warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      const uint8_t* sfa = p.sfa + static_cast<int64_t>(row0 >> 7) * p.tiles_k * 512;
      const uint8_t* sfb = p.sfb + static_cast<int64_t>(n0 >> 7) * p.tiles_k * 512;
      bool ok = true;
#pragma unroll 1
      for (int kb = first; kb < kb1; ++kb) {
        const int i = kb - first, stage = i % STAGES;
        if (!wait_or_abort(&empty_bar[stage], ((i / STAGES) & 1) ^ 1u, abort_flag)) {
          report_timeout(p.status, 1, 1); *abort_flag = 1; ok = false;
          break;
        }
        uint8_t* a_s = smem + stage * L::kOperand;
        if (kb < kb0) {
          mbar_arrive_expect_tx(&full_bar[stage], static_cast<uint32_t>(p.a_rows * BK + L::kBBytes));
          tma_load_2d(a_s, &tmT, &full_bar[stage], 0, row0);
          tma_load_2d(a_s + L::kABytes, &tmLb, &full_bar[stage], 0, n0);
          continue;
        }
        uint8_t* s_s = smem + L::kScaleOff + stage * 2 * L::kScale;
        const int t0 = kb * F::kTilesPerStage;
        const uint32_t sbytes = static_cast<uint32_t>(p.tiles_k - t0 < F::kTilesPerStage ? p.tiles_k - t0 : F::kTilesPerStage) * 512u;
        mbar_arrive_expect_tx(&full_bar[stage], static_cast<uint32_t>(p.a_rows * BK + L::kBBytes) + 2 * sbytes);
        tma_load_2d(a_s, &tmA, &full_bar[stage], kb * BK, row0);
        tma_load_2d(a_s + L::kABytes, &tmW, &full_bar[stage], kb * BK, n0);
        bulk_load(s_s, sfa + static_cast<int64_t>(t0) * 512, sbytes, &full_bar[stage]);
        bulk_load(s_s + L::kScale, sfb + static_cast<int64_t>(t0) * 512, sbytes, &full_bar[stage]);
      }
      if (!ok)                                          // copies in flight must land before the CTA may exit
        for (int k = 0; k < 64; ++k) __nanosleep(1000);
    }
  } else if (aligned_ok && warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      // columns [64, 128) of a weight row group start two scale words further on
      const uint32_t sfb_shift = static_cast<uint32_t>((n0 & 64) >> 5);
      bool ok = true;
#pragma unroll 1
      for (int kb = first; kb < kb1; ++kb) {
        const int i = kb - first, stage = i % STAGES;
        if (!wait_or_abort(&full_bar[stage], (i / STAGES) & 1, abort_flag)) {
          report_timeout(p.status, 2, 1); *abort_flag = 1; ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(smem + stage * L::kOperand);
        const uint64_t a_desc = make_kmajor_sw128_desc(a_addr);
        const uint64_t b_desc = make_kmajor_sw128_desc(a_addr + L::kABytes);
        if (kb < kb0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma_tf32(tmem_base, a_desc + static_cast<uint64_t>(2 * j), b_desc + static_cast<uint64_t>(2 * j), make_idesc_tf32(BM, BN),
                        j > 0 ? 1u : 0u);
          tc_commit(&empty_bar[stage]);
          // the accumulator is whole before the other kind of MMA adds to it; the first use of the first stage
          if (!wait_or_abort(&empty_bar[stage], 0u, abort_flag)) {
            report_timeout(p.status, 2, 4); *abort_flag = 1; ok = false;
            break;
          }
          tc_fence_after();
          continue;
        }
        const uint32_t s_addr = smem_u32(smem + L::kScaleOff + stage * 2 * L::kScale);
        const uint32_t sfa_t = tmem_base + BN + stage * L::kSetCols;
        const uint32_t sfb_t = sfa_t + 4 * F::kTilesPerStage;
        const int left = p.K - kb * kFp4StageK;                      // elements of this stage and beyond
#pragma unroll
        for (int j = 0; j < F::kTilesPerStage; ++j) {
          if (j * F::kTileK < left) {
            tc_cp_scale_tile(sfa_t + 4 * j, scale_tile_desc(s_addr + j * 512));
            tc_cp_scale_tile(sfb_t + 4 * j, scale_tile_desc(s_addr + L::kScale + j * 512));
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j * 64 < left) {
            const int t = j * 64 / F::kTileK;
            const uint32_t idesc = make_idesc_fp4(BM, BN, FMT == PQ_FP4_MX, FMT == PQ_FP4_MX ? 2 * (j & 1) : 0);
            tc_mma_fp4<FMT>(tmem_base, a_desc + static_cast<uint64_t>(2 * j), b_desc + static_cast<uint64_t>(2 * j), idesc,
                            sfa_t + 4 * t, sfb_t + 4 * t + sfb_shift, (i > 0 || j > 0) ? 1u : 0u);
          }
        }
        tc_commit(&empty_bar[stage]);
      }
      if (ok) tc_commit(done_bar);
    }
  } else if (aligned_ok) {
    // ------------------------------------------------------------------ epilogue
    const int et = threadIdx.x - 64;
    if (et < BN) {
      const int n = n0 + et;
      col_scale[et] = (p.s_col != nullptr && n < p.N) ? p.s_col[n] : 1.0f;
      col_bias[et] = (p.bias != nullptr && n < p.N) ? p.bias[n] : 0.0f;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int row = row0 + r;
    const float s_row = (p.s_row != nullptr && row < p.M) ? p.s_row[row] : 1.0f;
    const bool landed = wait_or_abort(done_bar, 0u, abort_flag);
    if (!__all_sync(0xffffffffu, landed)) {
      report_timeout(p.status, 3, 2); *abort_flag = 1;
    } else {
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tmem_base + c + (static_cast<uint32_t>(quarter * 32) << 16), v);
        tc_wait_ld();
        if constexpr (SPLIT) {
          if (row < p.M) {
            float* red = reinterpret_cast<float*>(smem) + r * L::kRedStride + c;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(red + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        } else {
          uint8_t* line = smem + r * L::kRowStride + 2 * c;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int i = 8 * j + 2 * k;
              w[k] = pack2_any(fmaf(__uint_as_float(v[i]), s_row * col_scale[c + i], col_bias[c + i]),
                               fmaf(__uint_as_float(v[i + 1]), s_row * col_scale[c + i + 1], col_bias[c + i + 1]), p.bf16);
            }
            *reinterpret_cast<uint4*>(line + 16 * j) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
    if constexpr (!SPLIT) {
      // every warp stores a quarter of the rows that there are, whole rows at a time; all reach this barrier, landed or not
      asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
      if (__all_sync(0xffffffffu, landed)) {
        unsigned short* const out = static_cast<unsigned short*>(p.out) + static_cast<int64_t>(row0) * p.ldo + n0;
        const int rows = p.M - row0 < BM ? p.M - row0 : BM;
        if (p.vec && n0 + BN <= p.N) {                     // four rows of eight 16-byte pieces
#pragma unroll 2
          for (int q = 4 * quarter + (lane >> 3); q < rows; q += 16)
            st_v4(out + q * p.ldo + (lane & 7) * 8, *reinterpret_cast<const uint4*>(smem + q * L::kRowStride + (lane & 7) * 16));
        } else {
#pragma unroll 2
          for (int q = quarter; q < rows; q += 4)
            store_row64(out + q * p.ldo, p.N - n0, lane, [&](int c) {
              return static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(smem + q * L::kRowStride + 2 * c));
            });
        }
      }
    }
    tc_fence_before();
  }

  __syncthreads();
  if constexpr (SPLIT) {
    // Partial tiles stand in the CTAs' shared memory; this CTA adds up its share of the 8-column pieces.  (Two columns a lane, so
    // that a warp stores whole rows, is slower for its four times as many reads: 64 x 10240 -> 2560 11.6 us instead of 10.7.)
    const bool ok = *abort_flag == 0;
    cluster_sync_all();
    if (ok) {
      const int rows = p.M - row0 < BM ? p.M - row0 : BM;
      const int items = rows * (BN / 8);
      const int per = (items + split - 1) / split;
      const int end = (rank + 1) * per < items ? (rank + 1) * per : items;
      for (int it = rank * per + static_cast<int>(threadIdx.x); it < end; it += kFp4Threads) {
        const int r = it / (BN / 8), c = it % (BN / 8) * 8;
        if (n0 + c >= p.N) continue;
        const uint32_t a = smem_u32(reinterpret_cast<float*>(smem) + r * L::kRedStride + c);
        float y[8] = {};
        for (int s = 0; s < split; ++s) {
          const uint32_t b = map_to_cta(a, static_cast<uint32_t>(s));
          const float4 u = ld_cluster_f4(b), w = ld_cluster_f4(b + 16);
          y[0] += u.x; y[1] += u.y; y[2] += u.z; y[3] += u.w;
          y[4] += w.x; y[5] += w.y; y[6] += w.z; y[7] += w.w;
        }
        const float s_row = p.s_row != nullptr ? p.s_row[row0 + r] : 1.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = fmaf(y[k], s_row * col_scale[c + k], col_bias[c + k]);
        store8(p, row0 + r, n0 + c, y);
      }
    }
    cluster_sync_all();                                  // peers read this CTA's shared memory until here
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, L::kTmemCols);
}

template <int FMT, int STAGES, bool SPLIT>
int launch_fp4(const CUtensorMap& tmA, const CUtensorMap& tmW, const CUtensorMap& tmT, const CUtensorMap& tmLb, const Fp4GemmParams& p, int split, cudaStream_t st) {
  using L = Fp4Smem<FMT, STAGES>;
  auto kern = pq_fp4_gemm_kernel<FMT, STAGES, SPLIT>;
  static bool attr_set[64] = {false};     // per device; benign race: the attribute value never changes
  int dev = 0;
  PQ_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    PQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.mt) * static_cast<unsigned>(p.nt) * static_cast<unsigned>(SPLIT ? split : 1));
  cfg.blockDim = dim3(kFp4Threads);
  cfg.dynamicSmemBytes = L::kTotal;
  cfg.stream = st;
  cudaLaunchAttribute at[2] = {chained_launch()};
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = static_cast<unsigned>(SPLIT ? split : 1);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = SPLIT ? 2 : 1;
  PQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tmA, tmW, tmT, tmLb, p, split));
  return PQ_OK;
}

template <int FMT>
int dispatch_fp4(const uint8_t* xq, int64_t ldx, const uint8_t* w, int64_t ldw, Fp4GemmParams& p, cudaStream_t st) {
  const int sms = sm_count();
  const int num_kb = (p.K + kFp4StageK - 1) / kFp4StageK;
  // 256 x 256 tiles on CTA pairs from a quarter of the SMs on, measured in us (mx, nv within 0.7), pair / single: 4096 x 640 -> 640
  // (48 tiles) 6.2 / 7.6, 1024 x 1280 -> 2560 (40) 7.2 / 9.3, -> 1920 (32) 7.2 / 6.2, -> 1280 (20) 7.2 / 5.9.  Up to 128 rows or
  // columns half a tile or more is unused: 128 x 1280 -> 10240 (40) 7.4 / 5.9, 128 x 4096 -> 32768 (128) 21.4 / 23.4;
  // 16384 x 640 -> 128 (64) 7.2 / 5.5, 65536 x 1280 -> 128 (256) 16.8 / 23.7, 65536 x 640 -> 64 12.7 / 8.9.
  const int64_t pair_tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + 255) / 256);
  const bool pair = p.N > 128 ? (p.M > 128 ? 4 : 2) * pair_tiles >= sms : (p.N > 64 && pair_tiles >= sms);
  if ((p.s_row != nullptr) == (p.s_col != nullptr) && (options().fp4_pair == 2 || (options().fp4_pair == 1 && pair)))
    return launch_fp4_pair(FMT, xq, ldx, w, ldw, p, st);
  p.nt = (p.N + BN - 1) / BN;
  const int64_t tiles = static_cast<int64_t>(p.mt) * p.nt;
  if (tiles > 0x0fffffff) return PQ_ERR_SHAPE;
  CUtensorMap tmA, tmW, tmT = {}, tmLb = {};
  // a single tile of few rows loads only those: what the others hold ends up in rows that nobody stores
  p.a_rows = p.M < BM ? (p.M + 7) / 8 * 8 : BM;
  int rc = make_tile_map(&tmA, xq, p.M, p.K / 2, ldx, p.a_rows);
  if (rc != PQ_OK) return rc;
  rc = make_tile_map(&tmW, w, p.N, p.K / 2, ldw, BN);
  if (rc != PQ_OK) return rc;
  if (p.t != nullptr && ((rc = make_tile_map(&tmT, p.t, p.M, BK, BK, p.a_rows)) != PQ_OK || (rc = make_tile_map(&tmLb, p.lb, p.N, BK, BK, BN)) != PQ_OK))
    return rc;
  // Along K a stage takes 0.26 us; a cluster costs 1 to 2 us, the more the more rows the joined tiles have, and runs in rounds when
  // the clusters do not all find room at once (2560 -> 2560, 40 tiles: 6.0 us split in two, 10.2 in four).  Measured in us,
  // unsplit / in two / in four, by stages: 77 rows -> 640 (10 tiles) 8 stages 5.5 / 6.6 / 6.5 (-> 1280), 10: 6.2 / 6.9 / 6.5,
  // 13: 6.9 / 7.2 / 6.5, 40: 13.7 / 10.6 / 8.6.  Where only two find room, 40 tiles of 16 rows 13: 6.9 / 6.9, 16: 7.6 / 6.9,
  // 50 tiles of 128 rows 16: 7.9 / 8.6, 20: 8.9 / 8.9, 40: 13.8 / 11.6.
  int split = 1;
  const bool only_two = tiles * 4 > sms * 3 / 4;
  if (num_kb >= (!only_two ? 10 : p.M <= 64 ? 14 : 20))
    while (split < 8 && tiles * split * 2 <= sms * 3 / 4 && split * 4 <= num_kb) split *= 2;
  const int want = options().fp4_split;
  if (want == 1 || want == 2 || want == 4 || want == 8) {
    split = want;
    while (split > num_kb) split /= 2;
  }
  if (split > 1) return launch_fp4<FMT, 7, true>(tmA, tmW, tmT, tmLb, p, split, st);
  if (tiles > sms) return launch_fp4<FMT, 3, false>(tmA, tmW, tmT, tmLb, p, 1, st);
  return launch_fp4<FMT, 7, false>(tmA, tmW, tmT, tmLb, p, 1, st);
}

}  // namespace
}  // namespace pq

using namespace pq;

extern "C" int pq_fp4_gemm_lowrank(const uint8_t* xq, int64_t ldx, const uint8_t* x_scales, const float* s_row, const uint8_t* w,
                                   int64_t ldw, const uint8_t* w_scales, const float* s_col, const float* bias, const float* t,
                                   const float* lb, int fmt, void* out, int out_dtype, int64_t ldo, int64_t M, int64_t N, int64_t K,
                                   void* workspace, size_t ws_bytes, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || M > 0x7fffff00LL || N > 0x7fffff00LL || K > 0x7fffff00LL) return PQ_ERR_SHAPE;
  if (out_dtype != PQ_DTYPE_BF16 && out_dtype != PQ_DTYPE_FP16) return PQ_ERR_DTYPE;
  if (fmt != PQ_FP4_MX && fmt != PQ_FP4_NV) return PQ_ERR_UNSUPPORTED;
  if (M == 0) return PQ_OK;
  if (xq == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || out == nullptr) return PQ_ERR_NULL;
  if ((t == nullptr) != (lb == nullptr)) return PQ_ERR_NULL;
  if (fmt == PQ_FP4_NV && (s_row == nullptr || s_col == nullptr)) return PQ_ERR_NULL;
  if (ldx < K / 2 || ldw < K / 2 || ldo < N) return PQ_ERR_SHAPE;
  if (K % 32 != 0 || ldx % 16 != 0 || ldw % 16 != 0) return PQ_ERR_ALIGN;
  if (!aligned_to(xq, 16) || !aligned_to(w, 16) || !aligned_to(x_scales, 16) || !aligned_to(w_scales, 16) || !aligned_to(out, 2) ||
      !aligned_to(s_row, 4) || !aligned_to(s_col, 4) || !aligned_to(bias, 4) || !aligned_to(t, 16) || !aligned_to(lb, 16))
    return PQ_ERR_ALIGN;
  if (workspace != nullptr && ws_bytes < PQ_GEMM_WORKSPACE_BYTES) return PQ_ERR_WORKSPACE;
  Fp4GemmParams p{};
  p.sfa = x_scales; p.sfb = w_scales; p.s_row = s_row; p.s_col = s_col; p.bias = bias; p.t = t; p.lb = lb; p.out = out;
  p.status = static_cast<int32_t*>(workspace);
  p.ldo = ldo; p.M = static_cast<int>(M); p.N = static_cast<int>(N); p.K = static_cast<int>(K);
  p.tiles_k = static_cast<int>(fp4_scale_tiles(K, fmt));
  p.mt = static_cast<int>((M + BM - 1) / BM);
  p.bf16 = out_dtype == PQ_DTYPE_BF16 ? 1 : 0;
  p.vec = ldo % 8 == 0 && aligned_to(out, 16) ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return fmt == PQ_FP4_MX ? dispatch_fp4<PQ_FP4_MX>(xq, ldx, w, ldw, p, st) : dispatch_fp4<PQ_FP4_NV>(xq, ldx, w, ldw, p, st);
}

extern "C" int pq_fp4_gemm(const uint8_t* xq, int64_t ldx, const uint8_t* x_scales, const float* s_row, const uint8_t* w,
                           int64_t ldw, const uint8_t* w_scales, const float* s_col, const float* bias, int fmt, void* out,
                           int out_dtype, int64_t ldo, int64_t M, int64_t N, int64_t K, void* workspace, size_t ws_bytes,
                           void* stream) {
  return pq_fp4_gemm_lowrank(xq, ldx, x_scales, s_row, w, ldw, w_scales, s_col, bias, nullptr, nullptr, fmt, out, out_dtype, ldo, M, N, K,
                             workspace, ws_bytes, stream);
}
