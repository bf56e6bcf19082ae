// Block-scaled 4-bit GEMM on CTA pairs (tcgen05 cta_group::2), the kernel of the large products; operands, scales and
// epilogue arithmetic as in gemm_fp4.cu.
//
// A cluster of two CTAs computes a 256 x 256 tile: CTA r owns rows [128 r, +128) of it in its own tensor memory, loads its
// own 128 activation rows and their scales, HALF of the weight rows, and all 256 rows of weight scales (each SM's tensor
// core needs them).  Per stage of K = 256 an SM pulls 32 KB of codes and 3 (mx) or 6 (nv) KB of scales from L2 for
// 512 cycles of MMA; the 128 x 128 tiles of the single-CTA kernel need 34 to 36 KB for 256 cycles.
//
// Tensor memory, 512 columns: two accumulators of 256 columns would leave no room for scales, so they overlap:
//   accumulator 0 [0, 256), accumulator 1 [128, 384), scale sets [384, 512).
// The epilogue of a tile drains the shared columns [128, 256) first and signals `shared_free`; then the next tile's MMAs
// may start in the other accumulator while the epilogue goes on with the columns that belong to its own alone.
// A scale set is written again only once the MMAs that read it have completed: with as many sets as stages (mx) the
// stage's own hand-over shows that; nv needs twice the columns, so its sets are those of half a stage, five of them, and
// before a stage the MMA thread waits for the first half of the stage before last, whose completion covers the last
// readers of both sets it is about to write.
//
// Warps: 0 TMA producer, 1 MMA issuer (leader CTA), 2-9 epilogue (a 32-row quarter and, step by step, 64 columns each:
// scale, bias, rounding, swizzled 4 KB staging block, TMA store; plain stores where TMA cannot address the rows).  Tiles go to the pairs in the order of blocks of eight
// row tiles, columns outside, so that the pairs at work share few activation and weight tiles.  Every wait is bounded; no
// multicast.
#include "gemm_fp4_common.cuh"

namespace pq {
namespace {

constexpr int kPairEpiWarps = 8;
constexpr int kPairThreads = (2 + kPairEpiWarps) * 32;
constexpr int kPairStages = 5;
constexpr int kRowBlock = 8;                     // row tiles per block of the tile order

template <int FMT>
struct Fp4PairSmem {
  static constexpr int kABytes = BM * BK, kBBytes = 128 * BK;
  static constexpr int kOperand = kABytes + kBBytes;
  static constexpr int kSfa = Fp4Fmt<FMT>::kScaleBytes, kSfb = 2 * Fp4Fmt<FMT>::kScaleBytes;
  static constexpr int kStageBytes = kOperand + kSfa + kSfb;                 // per CTA
  static constexpr int kOutOff = kPairStages * kOperand;                     // 1024-byte aligned blocks first
  static constexpr int kOutBlock = 32 * 128;
  static constexpr int kScaleOff = kOutOff + kPairEpiWarps * kOutBlock;
  static constexpr int kColOff = kScaleOff + kPairStages * (kSfa + kSfb);    // {scale, bias} of 256 columns, two tiles
  static constexpr int kBarOff = kColOff + 2 * 256 * 8;
  static constexpr int kNumBars = 3 * kPairStages + 2;                       // full, empty, acc_full, shared_free, half
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kTotal = kMiscOff + 16;
  static_assert(kTotal <= 232448, "exceeds the 227 KB shared memory of one CTA");
  // scale columns are handed over in units of a stage (mx) or half a stage (nv): per scale tile 4 columns for A, 8 for B
  static constexpr int kUnits = FMT == PQ_FP4_MX ? 1 : 2;
  static constexpr int kTilesPerUnit = Fp4Fmt<FMT>::kTilesPerStage / kUnits;
  static constexpr int kSetCols = 12 * kTilesPerUnit;
  static constexpr int kSets = 5;
  static_assert(384 + kSets * kSetCols <= 512, "tensor memory");
};

// scale tiles: three-dimensional TMA load {word, scale tile, row group}, zero-filled past the ends
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* m, uint32_t bar_cluster_addr, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(m), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
      : "memory");
}
template <int FMT>
__device__ __forceinline__ void tc_mma_fp4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa_tmem,
                                                uint32_t sfb_tmem, uint32_t acc) {
  if constexpr (FMT == PQ_FP4_MX)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(acc)
        : "memory");
}
// both CTAs copy the tile at this offset of their own shared memory into their own tensor memory
__device__ __forceinline__ void tc_cp_scale_tile_pair(uint32_t tmem_addr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem_addr), "l"(desc) : "memory");
}

// a load that stays where it is written (the compiler would move an ordinary one down to its use)
__device__ __forceinline__ float ld_now(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// Tile order: blocks of kRowBlock row tiles, inside a block column after column, rows innermost.  A pair visits every
// `stride`-th tile; the step needs no division (two of them took a third of the epilogue's time per tile) except in a last
// block of fewer rows.
struct Fp4PairWalker {
  int t, stride, tiles, nt_total, mt_total;
  int block_t0, block_row0;             // first tile and first row tile of the current block
  int mt, nt;                           // row tile, column tile
  __device__ __forceinline__ void init(int pair, int pairs, int mt_total_, int nt_total_) {
    t = pair; stride = pairs; mt_total = mt_total_; nt_total = nt_total_; tiles = mt_total * nt_total;
    block_t0 = block_row0 = 0;
    place();
  }
  __device__ __forceinline__ bool valid() const { return t < tiles; }
  __device__ __forceinline__ void place() {
    if (t >= tiles) return;
    const int full = kRowBlock * nt_total;
    while (t - block_t0 >= full) { block_t0 += full; block_row0 += kRowBlock; }
    const int rem = t - block_t0, left = mt_total - block_row0;
    nt = left >= kRowBlock ? rem / kRowBlock : rem / left;
    mt = block_row0 + rem - nt * (left >= kRowBlock ? kRowBlock : left);
  }
  __device__ __forceinline__ void advance() { t += stride; place(); }
};

template <int FMT, bool SCALED, typename OutT>
__global__ void __launch_bounds__(kPairThreads, 1)
pq_fp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                        const __grid_constant__ CUtensorMap tmSa, const __grid_constant__ CUtensorMap tmSw,
                        const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmT,
                        const __grid_constant__ CUtensorMap tmLb, const Fp4GemmParams p) {
  using L = Fp4PairSmem<FMT>;
  using F = Fp4Fmt<FMT>;
  constexpr int S = kPairStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty_bar = full_bar + S;
  uint64_t* acc_full = empty_bar + S;
  uint64_t* shared_free = acc_full + 1;
  uint64_t* half_bar = shared_free + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank();
  const bool aligned_ok = (smem_u32(smem) & 1023u) == 0;
  const int pair = static_cast<int>(blockIdx.x) >> 1, pairs = static_cast<int>(gridDim.x) >> 1;
  const int tiles = p.mt * p.nt;                                   // of 256 x 256
  const int num_kb = (p.K + kFp4StageK - 1) / kFp4StageK;
  const bool low = p.t != nullptr;                                 // a stage of its own in front of each tile's

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmW); tma_prefetch_desc(&tmSa); tma_prefetch_desc(&tmSw);
    if (p.vec) tma_prefetch_desc(&tmOut);
    for (int s = 0; s < S; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(acc_full, 1); mbar_init(shared_free, 2 * kPairEpiWarps);
    for (int s = 0; s < S; ++s) mbar_init(&half_bar[s], 1);
    *abort_flag = aligned_ok ? 0 : 1;
    if (!aligned_ok) report_timeout(p.status, 7, 7);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) { tmem_alloc_pair(tmem_holder, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                 // both CTAs' barriers exist before anyone signals across the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  wait_for_previous_kernel();         // (the next kernel is not let in early: 16384 x 1280 -> 1280 and its quantisation 29.0 us, 32.1 if so)
  auto leader_addr = [&](const uint64_t* bar) { return map_to_cta(smem_u32(bar), 0u); };
  auto peer_addr = [&](const uint64_t* bar) { return map_to_cta(smem_u32(bar), 1u); };

  if (aligned_ok && warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      int stage = 0; uint32_t phase = 0; int issued = 0; bool ok = true;
      Fp4PairWalker w; w.init(pair, pairs, p.mt, p.nt);
#pragma unroll 1
      for (; w.valid() && ok; w.advance()) {
        const int row0 = w.mt * 256 + static_cast<int>(rank) * BM;
        const int n0 = w.nt * 256;
        const int nhalf0 = n0 + static_cast<int>(rank) * 128;
#pragma unroll 1
        for (int kb = low ? -1 : 0; kb < num_kb; ++kb) {
          if (!wait_or_abort(&empty_bar[stage], phase ^ 1u, abort_flag)) {
            report_timeout(p.status, 1, 1); *abort_flag = 1; ok = false; break;
          }
          uint8_t* a_s = smem + stage * L::kOperand;
          uint8_t* s_s = smem + L::kScaleOff + stage * (L::kSfa + L::kSfb);
          const uint32_t fb = leader_addr(&full_bar[stage]);
          if (kb < 0) {
            if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * L::kOperand);
            tma_load_2d_pair(a_s, &tmT, fb, 0, row0);
            tma_load_2d_pair(a_s + L::kABytes, &tmLb, fb, 0, nhalf0);
          } else {
            if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * L::kStageBytes);
            tma_load_2d_pair(a_s, &tmA, fb, kb * BK, row0);
            tma_load_2d_pair(a_s + L::kABytes, &tmW, fb, kb * BK, nhalf0);
            tma_load_3d_pair(s_s, &tmSa, fb, 0, kb * F::kTilesPerStage, row0 >> 7);
            tma_load_3d_pair(s_s + L::kSfa, &tmSw, fb, 0, kb * F::kTilesPerStage, n0 >> 7);
          }
          if (issued < S) ++issued;
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
      // copies in flight must land before the CTA may exit: the last stages issued are consumed by MMAs whose
      // completion is committed to this CTA's empty barriers
      for (int i = 0; i < issued; ++i) {
        if (--stage < 0) { stage = S - 1; phase ^= 1u; }
        if (!wait_or_abort(&empty_bar[stage], phase, abort_flag)) {
          for (int k = 0; k < 64; ++k) __nanosleep(1000);
          break;
        }
      }
    }
  } else if (aligned_ok && warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issuer (leader CTA only)
    if (elect_one()) {
      int stage = 0; uint32_t phase = 0; int it = 0; bool ok = true;
      uint32_t set = 0; int issued = 0;                    // next scale set; stages issued (up to 2)
      auto commit_both = [&](uint64_t* bar) { tc_commit_pair(smem_u32(bar)); tc_commit_pair(peer_addr(bar)); };
      // Barriers are probed one step ahead of their use: a probe takes a few hundred cycles while the tensor cores and TMA
      // saturate shared memory, as long as a stage's MMAs.
      bool full_ready = false;
#pragma unroll 1
      for (int t = pair; t < tiles && ok; t += pairs, ++it) {
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>((it & 1) * 128);
        uint64_t* low_done = nullptr; uint32_t low_phase = 0;
        if (low) {
          if (!full_ready && !wait_or_abort(&full_bar[stage], phase, abort_flag)) {
            report_timeout(p.status, 2, 1); *abort_flag = 1; ok = false; break;
          }
          if (it > 0 && !wait_or_abort(shared_free, static_cast<uint32_t>(it - 1) & 1u, abort_flag)) {
            report_timeout(p.status, 2, 2); *abort_flag = 1; ok = false; break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + stage * L::kOperand);
          const uint64_t a_desc = make_kmajor_sw128_desc(a_addr), b_desc = make_kmajor_sw128_desc(a_addr + L::kABytes);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma_tf32_pair(d_tmem, a_desc + static_cast<uint64_t>(2 * j), b_desc + static_cast<uint64_t>(2 * j),
                             make_idesc_tf32(2 * BM, 256), j > 0 ? 1u : 0u);
          // this stage has no scales; the hand-over of scale sets counts it all the same
          if (L::kUnits > 1) tc_commit_pair(smem_u32(&half_bar[stage]));
          if (issued < 2) ++issued;
          commit_both(&empty_bar[stage]);
          low_done = &empty_bar[stage]; low_phase = phase;
          full_ready = false;
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
#pragma unroll 1
        for (int kb = 0; kb < num_kb && ok; ++kb) {
          // nv: the scale columns of this stage were last read by MMAs up to the first half of the stage before last
          if (L::kUnits > 1 && issued >= 2) {
            const int back = stage >= 2 ? stage - 2 : stage - 2 + S;
            if (!wait_or_abort(&half_bar[back], stage >= 2 ? phase : phase ^ 1u, abort_flag)) {
              report_timeout(p.status, 2, 3); *abort_flag = 1; ok = false; break;
            }
          }
          if (issued < 2) ++issued;
          if (!full_ready && !wait_or_abort(&full_bar[stage], phase, abort_flag)) {
            report_timeout(p.status, 2, 1); *abort_flag = 1; ok = false; break;
          }
          tc_fence_after();
          const int next = stage + 1 == S ? 0 : stage + 1;
          full_ready = mbar_test_wait(&full_bar[next], next == 0 ? phase ^ 1u : phase);
          const uint32_t a_addr = smem_u32(smem + stage * L::kOperand);
          const uint32_t s_addr = smem_u32(smem + L::kScaleOff + stage * (L::kSfa + L::kSfb));
          const uint64_t a_desc = make_kmajor_sw128_desc(a_addr);
          const uint64_t b_desc = make_kmajor_sw128_desc(a_addr + L::kABytes);
          const int left = p.K - kb * kFp4StageK;
#pragma unroll
          for (int u = 0; u < L::kUnits; ++u) {
            const uint32_t sfa_t = tmem_base + 384 + set * L::kSetCols;
            const uint32_t sfb_t = sfa_t + 4 * L::kTilesPerUnit;
#pragma unroll
            for (int j = 0; j < L::kTilesPerUnit; ++j) {
              const int tile = u * L::kTilesPerUnit + j;
              tc_cp_scale_tile_pair(sfa_t + 4 * j, scale_tile_desc(s_addr + tile * 512));
              tc_cp_scale_tile_pair(sfb_t + 8 * j, scale_tile_desc(s_addr + L::kSfa + tile * 512));
              tc_cp_scale_tile_pair(sfb_t + 8 * j + 4, scale_tile_desc(s_addr + L::kSfa + (F::kTilesPerStage + tile) * 512));
            }
            // The scales of a tile's first stage are under way before the accumulator is free, or before the low-rank term is whole
            // and the other kind of MMA may add to it (its stage is not used again before this thread goes on, so the barrier
            // keeps the parity waited for).
            if (u == 0 && kb == 0 && low) {
              if (!wait_or_abort(low_done, low_phase, abort_flag)) {
                report_timeout(p.status, 2, 4); *abort_flag = 1; ok = false; break;
              }
              tc_fence_after();
            } else if (u == 0 && kb == 0 && it > 0) {
              if (!wait_or_abort(shared_free, static_cast<uint32_t>(it - 1) & 1u, abort_flag)) {
                report_timeout(p.status, 2, 2); *abort_flag = 1; ok = false; break;
              }
              tc_fence_after();
            }
#pragma unroll
            for (int m = 0; m < 4 / L::kUnits; ++m) {
              const int j = u * (4 / L::kUnits) + m;
              if (j * 64 < left) {
                const int s = m * 64 / F::kTileK;
                const uint32_t idesc = make_idesc_fp4(2 * BM, 256, FMT == PQ_FP4_MX, FMT == PQ_FP4_MX ? 2 * (j & 1) : 0);
                tc_mma_fp4_pair<FMT>(d_tmem, a_desc + static_cast<uint64_t>(2 * j), b_desc + static_cast<uint64_t>(2 * j), idesc,
                                     sfa_t + 4 * s, sfb_t + 8 * s, (kb > 0 || j > 0 || low) ? 1u : 0u);
              }
            }
            if (L::kUnits > 1 && u == 0) tc_commit_pair(smem_u32(&half_bar[stage]));
            if (++set == L::kSets) set = 0;
          }
          if (!ok) break;
          commit_both(&empty_bar[stage]);
          if (next == 0) phase ^= 1u;
          stage = next;
        }
        if (!ok) break;
        commit_both(acc_full);
      }
    }
  } else if (aligned_ok && warp >= 2) {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3, h = (warp - 2) >> 2, et = static_cast<int>(threadIdx.x) - 64;
    uint8_t* block = smem + L::kOutOff + (warp - 2) * L::kOutBlock;
    const int g = lane >> 2, q = lane & 3;       // accumulator fragments: rows g, g + 8 (+ 16), column pairs 8 j + 2 q
    const uint32_t block_addr = smem_u32(block) + g * 128 + q * 4;
    // A tile's column scales, bias and row scales are requested one tile ahead: in front of the accumulator's barrier their
    // latency would be paid on every tile.
    float next_scale = 1.0f, next_bias = 0.0f;
    float next_row[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    Fp4PairWalker w; w.init(pair, pairs, p.mt, p.nt);
    auto request = [&]() {
      if (!w.valid()) return;
      // indices are clamped, not tested: branches one after the other cost as much as the tile's conversion
      const int n = min(w.nt * 256 + et, p.N - 1), row = w.mt * 256 + static_cast<int>(rank) * BM + quarter * 32 + g;
      if (p.bias != nullptr) next_bias = ld_now(p.bias + n);
      if constexpr (SCALED) {
        next_scale = ld_now(p.s_col + n);
#pragma unroll
        for (int r = 0; r < 4; ++r) next_row[r] = ld_now(p.s_row + min(row + 8 * r, p.M - 1));
      }
    };
    request();
    int it = 0;
    bool ok = true;                     // after a wait that gave up a warp only keeps the column barriers' company
#pragma unroll 1
    for (; w.valid(); ++it) {
      const int row0 = w.mt * 256 + static_cast<int>(rank) * BM + quarter * 32;
      const int n0 = w.nt * 256;
      // {scale, scale, bias, bias} of column pairs, two buffers: the one written here was last read two tiles ago, before the
      // barrier of the last tile
      float* cols = reinterpret_cast<float*>(smem + L::kColOff) + (it & 1) * 512;
      cols[(et >> 1) * 4 + (et & 1)] = next_scale;
      cols[(et >> 1) * 4 + 2 + (et & 1)] = next_bias;
      float s_row[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) s_row[r] = next_row[r];
      asm volatile("bar.sync 1, %0;" ::"n"(kPairEpiWarps * 32) : "memory");
      w.advance();
      request();
      if (!ok) continue;
      const int buf = it & 1;
#pragma unroll 1
      for (int step = 0; step < 2; ++step) {
        // columns shared with the other accumulator first: the upper half of accumulator 0, the lower of accumulator 1
        const int c0 = ((buf ^ step) == 0 ? 128 : 0) + h * 64;
        float4 sb[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sb[j] = *reinterpret_cast<const float4*>(&cols[(c0 + 8 * j + 2 * q) * 2]);
        if (step == 0) {
          const bool landed = wait_or_abort(acc_full, static_cast<uint32_t>(it) & 1u, abort_flag);
          if (!__all_sync(0xffffffffu, landed)) { report_timeout(p.status, 3, 2); *abort_flag = 1; ok = false; break; }
          tc_fence_after();
        }
        uint32_t v[2][32];
        const uint32_t src = tmem_base + static_cast<uint32_t>(buf * 128 + c0) + (static_cast<uint32_t>(quarter * 32) << 16);
        tmem_ld_16x256b_x8(src, v[0]);
        tmem_ld_16x256b_x8(src + (16u << 16), v[1]);
        tc_wait_ld();
        if (step == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(leader_addr(shared_free));
        }
        if (lane == 0) bulk_wait_group_read0();               // the staging block's last store has been read
        __syncwarp();
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float2 y = make_float2(__uint_as_float(v[half][4 * j + 2 * r]), __uint_as_float(v[half][4 * j + 2 * r + 1]));
              const float2 b = make_float2(sb[j].z, sb[j].w);
              if constexpr (SCALED) {
                const float sr = s_row[2 * half + r];
                y = __ffma2_rn(y, __fmul2_rn(make_float2(sb[j].x, sb[j].y), make_float2(sr, sr)), b);
              } else {
                y = __fadd2_rn(y, b);
              }
              // row 16 half + 8 r + g of the block, 16-byte chunk j at its swizzled place: a warp's words fall into 32 banks
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(block_addr + (16 * half + 8 * r) * 128 + ((j ^ g) << 4)),
                           "r"(pack2(y.x, y.y, OutT{}))
                           : "memory");
            }
        if (p.vec) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && n0 + c0 < p.N && row0 < p.M) tma_store_2d(&tmOut, block, n0 + c0, row0);
          if (lane == 0) bulk_commit_group();
        } else {
          // rows that TMA cannot address (it stores 16 bytes at a time): the block's rows, 32 elements per instruction
          __syncwarp();
#pragma unroll 1
          for (int r = 0; r < 32 && row0 + r < p.M; ++r) {
            unsigned short* o = static_cast<unsigned short*>(p.out) + static_cast<int64_t>(row0 + r) * p.ldo + n0 + c0;
#pragma unroll
            for (int c = lane; c < 64; c += 32)
              if (n0 + c0 + c < p.N) o[c] = *reinterpret_cast<const unsigned short*>(block + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_group0();
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync_all();                 // neither CTA leaves while its peer may still signal it or read its shared memory
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// scale tiles as words: [row groups][tiles][128], box {128, tiles of a stage, groups}
int make_scale_map(CUtensorMap* map, const void* base, int64_t rows, int tiles, int box_tiles, int box_groups) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return PQ_ERR_CUDA;
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(tiles), static_cast<cuuint64_t>((rows + 127) / 128)};
  cuuint64_t strides[2] = {512, static_cast<cuuint64_t>(tiles) * 512};
  cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_tiles), static_cast<cuuint32_t>(box_groups)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { g_last_cuda_error = static_cast<int>(r); return PQ_ERR_CUDA; }
  return PQ_OK;
}
// output rows, box 64 columns x 32 rows, 128-byte swizzle; what lies past M or N is not written
int make_out_map(CUtensorMap* map, const void* base, int64_t M, int64_t N, int64_t ldo) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return PQ_ERR_CUDA;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ldo) * 2};
  cuuint32_t box[2] = {64, 32};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { g_last_cuda_error = static_cast<int>(r); return PQ_ERR_CUDA; }
  return PQ_OK;
}

template <int FMT, bool SCALED, typename OutT>
int launch_pair(const uint8_t* xq, int64_t ldx, const uint8_t* w, int64_t ldw, Fp4GemmParams p, cudaStream_t st) {
  using L = Fp4PairSmem<FMT>;
  using F = Fp4Fmt<FMT>;
  p.mt = (p.M + 255) / 256;
  p.nt = (p.N + 255) / 256;
  const int64_t tiles = static_cast<int64_t>(p.mt) * p.nt;
  if (tiles > 0x3fffffff) return PQ_ERR_SHAPE;
  p.vec = p.vec && p.N % 8 == 0;
  CUtensorMap tmA, tmW, tmSa, tmSw, tmOut = {}, tmT = {}, tmLb = {};
  int rc;
  if ((rc = make_tile_map(&tmA, xq, p.M, p.K / 2, ldx, BM)) != PQ_OK || (rc = make_tile_map(&tmW, w, p.N, p.K / 2, ldw, 128)) != PQ_OK ||
      (rc = make_scale_map(&tmSa, p.sfa, p.M, p.tiles_k, F::kTilesPerStage, 1)) != PQ_OK ||
      (rc = make_scale_map(&tmSw, p.sfb, p.N, p.tiles_k, F::kTilesPerStage, 2)) != PQ_OK ||
      (p.vec && (rc = make_out_map(&tmOut, p.out, p.M, p.N, p.ldo)) != PQ_OK) ||
      (p.t != nullptr && ((rc = make_tile_map(&tmT, p.t, p.M, BK, BK, BM)) != PQ_OK || (rc = make_tile_map(&tmLb, p.lb, p.N, BK, BK, 128)) != PQ_OK)))
    return rc;
  auto kern = pq_fp4_gemm_pair_kernel<FMT, SCALED, OutT>;
  static bool attr_set[64] = {false};     // per device; benign race: the attribute value never changes
  int dev = 0;
  PQ_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    PQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int pairs = sm_count() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2u * static_cast<unsigned>(tiles < pairs ? tiles : pairs));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = L::kTotal;
  cfg.stream = st;
  cudaLaunchAttribute at[2] = {chained_launch()};
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  PQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tmA, tmW, tmSa, tmSw, tmOut, tmT, tmLb, p));
  return PQ_OK;
}

template <typename OutT>
int launch_pair_as(int fmt, const uint8_t* xq, int64_t ldx, const uint8_t* w, int64_t ldw, const Fp4GemmParams& p, cudaStream_t st) {
  if (fmt == PQ_FP4_NV) return launch_pair<PQ_FP4_NV, true, OutT>(xq, ldx, w, ldw, p, st);
  if (p.s_row != nullptr) return launch_pair<PQ_FP4_MX, true, OutT>(xq, ldx, w, ldw, p, st);
  return launch_pair<PQ_FP4_MX, false, OutT>(xq, ldx, w, ldw, p, st);
}

}  // namespace

int launch_fp4_pair(int fmt, const uint8_t* xq, int64_t ldx, const uint8_t* w, int64_t ldw, const Fp4GemmParams& p, cudaStream_t st) {
  return p.bf16 ? launch_pair_as<__nv_bfloat16>(fmt, xq, ldx, w, ldw, p, st) : launch_pair_as<__half>(fmt, xq, ldx, w, ldw, p, st);
}

}  // namespace pq
