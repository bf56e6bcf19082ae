// Device helpers of the 4-bit floating-point path: E2M1 codes with one scale per block of elements.
//
// Arithmetic contract (x: 16-bit values, exact in fp32)
//   mx, blocks of 32:  s = 2^(floor(log2 max|x|) - 2), not below 2^-127, kept as an E8M0 byte (exponent + 127);
//   nv, blocks of 16:  s_row = the smallest power of two, not below 2^-100, with max|x over the row| <= 6 * 448 * s_row
//                      (1 for a row of zeros);  s = e4m3(max|x over the block| / (6 * s_row)), round half to even;
//   code = e2m1(x / s), e2m1(x / (s * s_row)): nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6, ties to the even code, larger
//   magnitudes to 6, the sign of x kept; an nv block whose s rounded to 0 gets codes 0.
// Every scale is exact or one rounding away from exact operands, and every quotient is either exact in fp32 or far from a
// rounding border of E2M1 compared with the fp32 rounding (x has at most 11 significant bits, border times scale at most
// 7), so fp32 gives the codes of exact arithmetic.
//   Not finite: an mx block with an infinity or a NaN gets the E8M0 NaN (255) and codes 0; an nv row gets s_row = NaN,
//   scales and codes 0.
//
// Scale bytes are laid out for tcgen05.cp (32x128b.warpx4): tiles of 128 rows x 4 consecutive scales, 512 bytes each,
// byte (r % 32) * 16 + (r / 32) * 4 + k of a tile = row r, scale k; tiles of one row group are consecutive.
#pragma once
#include "common.cuh"
#include "quant_common.cuh"

namespace pq {
namespace {

// Chained launches.  The kernels that take or make 4-bit rows follow one another on a stream, a few microseconds each, so they are
// launched with programmatic serialisation: a kernel's blocks may become resident, set up barriers and tensor memory and fetch
// descriptors while the kernel before it is still at work.  Every thread then waits for the end of that kernel, memory included,
// before its first access to global memory, so that nothing is read or overwritten early; a chain of such kernels waits link by
// link, as no block ends before its own wait.  Their loads are no read-only ones, which might be asked for ahead of the wait.
// Quantisation and product, us, plain launches / chained: 1 x 1280 -> 1280 6.6 / 5.7, 77 x 1280 -> 640 7.9 / 6.5, 4096 x 640 -> 640
// 10.1 / 9.1, 16384 x 1280 -> 1280 31.0 / 29.0.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// once all blocks have said so (or ended) the next kernel's may take what room is left
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
inline cudaLaunchAttribute chained_launch() {
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  return at;
}

// scale tiles per row group of 128 rows
__host__ __device__ __forceinline__ int64_t fp4_scale_tiles(int64_t K, int fmt) {
  const int64_t per = fmt == PQ_FP4_MX ? 128 : 64;                 // elements per four scales
  return (K + per - 1) / per;
}
// byte offset of scale tile `kt` of row `m` inside the scale array, at the row's first scale of that tile
__device__ __forceinline__ int64_t fp4_scale_off(int64_t m, int64_t kt, int64_t tiles) {
  return ((m >> 7) * tiles + kt) * 512 + (m & 31) * 16 + ((m >> 5) & 3) * 4;
}

// 32 contiguous, 32-byte aligned bytes (16 elements of 16 bits)
struct Chunk16 { uint32_t w[8]; };
__device__ __forceinline__ Chunk16 ld_stream_chunk16(const void* p) {
  Chunk16 c;
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(c.w[0]), "=r"(c.w[1]), "=r"(c.w[2]), "=r"(c.w[3]), "=r"(c.w[4]), "=r"(c.w[5]), "=r"(c.w[6]), "=r"(c.w[7])
               : "l"(p) : "memory");
  return c;
}
__device__ __forceinline__ void st_chunk16(void* p, const Chunk16& c) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(c.w[0]), "r"(c.w[1]), "r"(c.w[2]), "r"(c.w[3]),
               "r"(c.w[4]), "r"(c.w[5]), "r"(c.w[6]), "r"(c.w[7])
               : "memory");
}

// running maximum of the magnitudes of 16 packed elements (two packed halfword maxima, see absmax_chunk)
__device__ __forceinline__ uint32_t absmax_chunk16(const Chunk16& c) {
  constexpr uint32_t kMag = 0x7FFF7FFFu;
  uint32_t a = __vimax3_u16x2(c.w[0] & kMag, c.w[1] & kMag, c.w[2] & kMag);
  uint32_t b = __vimax3_u16x2(c.w[3] & kMag, c.w[4] & kMag, c.w[5] & kMag);
  return __vimax3_u16x2(__vimax3_u16x2(a, c.w[6] & kMag, c.w[7] & kMag), b, b);
}

// the larger of the two magnitudes, as a bit pattern (a maximum of floats would drop a NaN)
__device__ __forceinline__ uint32_t max_pattern(uint32_t acc) { return max(acc & 0xFFFFu, acc >> 16); }

// eight fp32 values -> eight E2M1 codes, element 0 in the low nibble of byte 0
__device__ __forceinline__ uint32_t pack_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// one byte of two codes per half: values as packed fp16 (exact)
__device__ __forceinline__ void unpack_e2m1x8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// non-negative fp32 -> E4M3 byte (round half to even, largest finite value beyond 448) and back
__device__ __forceinline__ uint32_t e4m3_of(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(byte)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xFFFFu)));
}

// s_row of an nv row from its largest magnitude (finite): 2688 = 1.3125 * 2^11
__device__ __forceinline__ float nv_row_scale(float amax) {
  const int bits = __float_as_int(amax);
  int e = (bits >> 23) - ((bits & 0x7FFFFF) <= 0x280000 ? 11 : 10);
  if (e < 27) e = 27;                                             // 2^-100
  return __int_as_float(bits == 0 ? 0x3F800000 : e << 23);
}

// Multiplier and divisor of one block.  code = e2m1(x / div): the quotient is estimated with the approximate reciprocal and
// corrected once.  With inv = (1 + e') / div and q0 = (1 + e) x / div, the corrected value is (1 - e e') x / div, e and e' below
// 2^-21, before its rounding: quotients that fp32 holds, the ties among them, come out exactly.  div == 0 marks a block of
// zero codes.
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
struct BlockScale { uint32_t byte; float inv, div; };
__device__ __forceinline__ BlockScale mx_block_scale(float amax) {
  BlockScale b;
  const int e = __float_as_int(amax) >> 23;
  b.byte = e == 255 ? 255u : (e > 2 ? static_cast<uint32_t>(e - 2) : 0u);
  b.inv = __int_as_float((254 - static_cast<int>(b.byte)) << 23);      // 2^(127 - byte); byte <= 252 when finite
  b.div = e == 255 ? 0.0f : 1.0f;                                       // power of two: the product is exact, no correction
  return b;
}
__device__ __forceinline__ BlockScale nv_block_scale(float amax, float s_row, bool bad_row) {
  BlockScale b;
  // amax / s_row is exact (power of two); the division by 6 rounds once, exact quotients (ties of E4M3 among them) exactly
  const float t = __fmul_rn(amax, __int_as_float(0x7F000000 - __float_as_int(s_row)));
  const float r6 = 0.16666667163372040f;                              // RN(1/6)
  const float q0 = __fmul_rn(t, r6);
  const float v = __fmaf_rn(__fmaf_rn(-q0, 6.0f, t), r6, q0);
  b.byte = bad_row ? 0u : e4m3_of(v);
  b.div = e4m3_value(b.byte) * s_row;
  b.inv = rcp_approx(b.div);
  if (bad_row) b.div = 0.0f;
  return b;
}

// mx: x / div; nv: -x / div, since the correction of x / div itself would make a negative zero positive (x - q0 div = +0, and
// +0 + -0 = +0) where that of the negative keeps both zeros' signs
template <int FMT>
__device__ __forceinline__ float2 e2m1_quotient(float2 x, const BlockScale& b) {
  if constexpr (FMT == PQ_FP4_MX) return __fmul2_rn(x, make_float2(b.inv, b.inv));
  const float2 ninv = make_float2(-b.inv, -b.inv);
  const float2 q0 = __fmul2_rn(x, ninv);
  return __ffma2_rn(__ffma2_rn(q0, make_float2(b.div, b.div), x), ninv, q0);
}

// 16 packed elements of one block (or half of an mx block) -> 8 bytes of codes
template <typename T, int FMT>
__device__ __forceinline__ uint2 quant_chunk16(const Chunk16& c, const BlockScale& b) {
  if (b.div == 0.0f) return make_uint2(0u, 0u);      // scale rounded to zero, or not finite
  uint2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = e2m1_quotient<FMT>(unpack2<T>(c.w[4 * h + i]), b);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
    (h == 0 ? r.x : r.y) = pack_e2m1x8(v) ^ (FMT == PQ_FP4_MX ? 0u : 0x88888888u);
  }
  return r;
}

}  // namespace
}  // namespace pq
