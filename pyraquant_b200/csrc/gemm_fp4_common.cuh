// Pieces shared by the block-scaled 4-bit GEMM kernels: parameters, the tcgen05 wrappers and descriptors of
// kind::mxf4 / kind::mxf4nvf4 and of the low-rank term.
//
// Operands.  A row of K E2M1 codes is K / 2 bytes, so a tile of 128-byte rows with the 128-byte swizzle holds 256
// elements per row and one MMA (K = 64) takes 32 bytes of it: the same bytes as an INT8 MMA of K = 32.
// Scales.  A scale tile (fp4_common.cuh) is exactly what tcgen05.cp.32x128b.warpx4 turns into four tensor-memory columns:
// 16 bytes per lane, word j of lane r = the four scales of row 32 j + r, replicated over the four lane quarters.  nv: a
// tile holds the scales of one MMA (4 x 16 elements).  mx: of two (2 x 32 elements each); the instruction descriptor's
// scale ids 0 and 2 pick the half.
#pragma once

#include "fp4_common.cuh"
#include "gemm_common.cuh"

namespace pq {

struct Fp4GemmParams {
  const uint8_t* sfa;      // scale tiles of the activations
  const uint8_t* sfb;      // and of the weights
  const float* s_row;      // [M] or NULL (1)
  const float* s_col;      // [N] or NULL (1)
  const float* bias;       // [N] or NULL
  const float* t;          // [M, 32] low-rank activations over s_row, or NULL
  const float* lb;         // [N, 32] low-rank up-projection over s_col
  void* out;
  int32_t* status;
  int64_t ldo;
  int M, N, K;
  int tiles_k;             // scale tiles per row group
  int mt, nt;              // row and column tiles
  int a_rows;              // rows of an activation tile that are loaded (single-CTA kernel)
  int bf16;                // output type
  int vec;                 // rows may be stored 16 bytes at a time
};

// The CTA-pair kernel (gemm_fp4_pair.cu): both row scales or neither.  Fills in the tile counts itself.
int launch_fp4_pair(int fmt, const uint8_t* xq, int64_t ldx, const uint8_t* w, int64_t ldw, const Fp4GemmParams& p, cudaStream_t st);

namespace {

constexpr int kFp4StageK = 256;                                   // elements per stage = 128 bytes

template <int FMT>
struct Fp4Fmt {
  static constexpr int kTilesPerStage = FMT == PQ_FP4_MX ? 2 : 4;       // scale tiles per stage and row group
  static constexpr int kTileK = kFp4StageK / kTilesPerStage;            // elements per scale tile
  static constexpr int kScaleBytes = kTilesPerStage * 512;
};

// Instruction descriptor of kind::mxf4 / kind::mxf4nvf4: E2M1 operands, K-major, shape M x N, scales E8M0 or E4M3.
__host__ __device__ constexpr uint32_t make_idesc_fp4(int M, int N, bool mx, int scale_id) {
  return (static_cast<uint32_t>(scale_id) << 4)                   // B scale id
         | (1u << 7)                                              // A format: E2M1
         | (1u << 10)                                             // B format: E2M1
         | (static_cast<uint32_t>(N >> 3) << 17)
         | ((mx ? 1u : 0u) << 23)                                 // scale format: E8M0 (else E4M3)
         | (static_cast<uint32_t>(M >> 4) << 24)
         | (static_cast<uint32_t>(scale_id) << 29);               // A scale id
}

// The low-rank term t @ lb^T is one more stage of the product, in front of the others: 32 fp32 values are 128 bytes, so its tiles are
// loaded, swizzled and addressed like those of 256 codes, and four kind::tf32 MMAs (K = 8) start the accumulator.  TF32 has the
// significand of fp16 and the exponents of fp32: 16-bit values over powers of two are exact in it.  The MMAs of the other kind
// are issued once these have completed.  Measured with the conversion of t, us, without the term / with it / with a library product
// added to the output instead: mx 77 x 2048 -> 1280 4.8 / 6.2 / 7.6, 16384 x 1280 -> 10240 100 / 119 / 249, 8192^3 186 / 195
// in short runs (power decides in long ones), 187 / 209 / 258 in long ones; nv 16384 x 1280 -> 1280 19.3 / 22.3 / 30.6.
__host__ __device__ constexpr uint32_t make_idesc_tf32(int M, int N) {
  return (1u << 4) | (2u << 7) | (2u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_tf32(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tc_mma_tf32_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}

template <int FMT>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa_tmem,
                                           uint32_t sfb_tmem, uint32_t acc) {
  if constexpr (FMT == PQ_FP4_MX)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(acc)
        : "memory");
}

// Shared-memory descriptor of a scale tile: 32 rows of 16 contiguous bytes, no swizzle, eight-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scale_tile_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}
__device__ __forceinline__ void tc_cp_scale_tile(uint32_t tmem_addr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem_addr), "l"(desc) : "memory");
}

// contiguous copy global -> shared, completion bytes on a barrier of this CTA; 16-byte aligned, size % 16 == 0
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ uint32_t pack2_any(float a, float b, int bf16) {
  return bf16 ? pack2(a, b, __nv_bfloat16{}) : pack2(a, b, __half{});
}

}  // namespace
}  // namespace pq
