// Quantisation of 16-bit rows to packed E2M1 codes with block scales, and the way back (formats and arithmetic:
// fp4_common.cuh).  HBM-bound: 2 bytes read, 0.53 (mx) or 0.56 (nv) written per element.
//
// A team of 8 to 256 threads owns a row.  A thread's unit is 16 contiguous elements, one 32-byte load and one 8-byte
// store of codes: an nv block is then one thread's, an mx block two neighbours', and the four scale bytes of a 32-bit
// word of the scale layout belong to four or eight neighbours and are joined by shuffles.  The nv row scale needs the
// whole row before the first code, so the row stays in registers (up to five units per thread) between the maximum and
// the codes; rows beyond 20480 elements are read twice.
#include "fp4_common.cuh"

namespace pq {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 5;                 // units of 16 elements a thread keeps in registers

template <int FMT>
__device__ __forceinline__ uint32_t join_scale_bytes(uint32_t byte, int lane_in_row) {
  // nv: lanes 4i .. 4i+3 hold scales 0 .. 3; mx: lanes 8i + 2k and 8i + 2k + 1 both hold scale k
  if constexpr (FMT == PQ_FP4_MX) {
    uint32_t w = byte << (8 * ((lane_in_row >> 1) & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 2);
    return w | __shfl_xor_sync(0xffffffffu, w, 4);
  } else {
    uint32_t w = byte << (8 * (lane_in_row & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    return w | __shfl_xor_sync(0xffffffffu, w, 2);
  }
}

// Codes and scales of one unit; every thread of a warp calls it (shuffles), units past the row's end with zeros.
template <typename T, int FMT>
__device__ __forceinline__ void quant_unit(const Chunk16& v, int c, int nchunk, bool row_ok, int64_t row, int lane_in_row,
                                           float s_row, bool bad_row, uint8_t* __restrict__ codes, int64_t row_bytes,
                                           uint8_t* __restrict__ scales, int64_t tiles) {
  constexpr int kPerWord = FMT == PQ_FP4_MX ? 8 : 4;                // units per four scales
  uint32_t m = max_pattern(absmax_chunk16(v));
  T tag{};
  BlockScale b;
  if constexpr (FMT == PQ_FP4_MX) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    b = mx_block_scale(lo_f32(m, tag));
  } else {
    b = nv_block_scale(lo_f32(m, tag), s_row, bad_row);
  }
  const uint32_t word = join_scale_bytes<FMT>(b.byte, lane_in_row);
  if (!row_ok) return;
  if (c < nchunk) {
    const uint2 q = quant_chunk16<T, FMT>(v, b);
    st_v2(codes + row * row_bytes + static_cast<int64_t>(c) * 8, q.x, q.y);
  }
  if (lane_in_row % kPerWord == 0 && c < nchunk)
    *reinterpret_cast<uint32_t*>(scales + fp4_scale_off(row, c / kPerWord, tiles)) = word;
}

// Largest magnitude of a row over its team; NaN and infinity come out as they order as bit patterns (above all finite).
template <typename T, int TPR>
__device__ __forceinline__ float team_amax(uint32_t acc, float* part, int tid) {
  uint32_t m = max_pattern(acc);
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if constexpr (TPR > 32) {
    uint32_t* p = reinterpret_cast<uint32_t*>(part);
    if ((tid & 31) == 0) p[tid >> 5] = m;
    __syncthreads();
    constexpr int WPR = TPR / 32;
    const int w0 = tid / TPR * WPR;
    m = p[w0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) m = max(m, p[w0 + w]);
  }
  T tag{};
  return lo_f32(m, tag);
}

template <typename T, int FMT, int TPR, bool LONG>
__global__ void __launch_bounds__(kThreads, LONG ? 2 : 3)
pq_quant_rows_fp4_kernel(const T* x, int64_t ldx, uint8_t* codes, uint8_t* scales, float* row_scale, int64_t M, int K) {
  constexpr int RPB = kThreads / TPR;
  __shared__ float part[kThreads / 32];
  wait_for_previous_kernel();
  allow_next_kernel();
  const int tid = threadIdx.x;
  const int lane = tid % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + tid / TPR;
  const bool row_ok = row < M;
  const int nchunk = K >> 4;
  const int64_t tiles = fp4_scale_tiles(K, FMT);
  const T* xrow = x + (row_ok ? row : 0) * ldx;
  const Chunk16 zero{};

  Chunk16 v[LONG ? 1 : kUnits];
  uint32_t acc = 0u;
  if constexpr (!LONG) {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int c = lane + j * TPR;
      v[j] = (row_ok && c < nchunk) ? ld_stream_chunk16(xrow + static_cast<int64_t>(c) * 16) : zero;
    }
  }
  float s_row = 1.0f;
  bool bad_row = false;
  if constexpr (FMT == PQ_FP4_NV) {
    if constexpr (LONG) {
      if (row_ok)
        for (int c = lane; c < nchunk; c += TPR) acc = __vimax3_u16x2(acc, acc, absmax_chunk16(ld_stream_chunk16(xrow + static_cast<int64_t>(c) * 16)));
    } else {
#pragma unroll
      for (int j = 0; j < kUnits; ++j) { const uint32_t a = absmax_chunk16(v[j]); acc = __vimax3_u16x2(acc, a, a); }
    }
    const float amax = team_amax<T, TPR>(acc, part, tid);
    bad_row = (__float_as_int(amax) >> 23) == 255;
    s_row = bad_row ? 1.0f : nv_row_scale(amax);
    if (row_ok && lane == 0) row_scale[row] = bad_row ? __int_as_float(0x7FC00000) : s_row;
  }
  const int64_t row_bytes = K >> 1;
  if constexpr (LONG) {
    for (int c0 = 0; c0 < nchunk; c0 += TPR) {
      const int c = c0 + lane;
      const Chunk16 u = (row_ok && c < nchunk) ? ld_stream_chunk16(xrow + static_cast<int64_t>(c) * 16) : zero;
      quant_unit<T, FMT>(u, c, nchunk, row_ok, row, lane, s_row, bad_row, codes, row_bytes, scales, tiles);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      if (j * TPR >= nchunk) break;                        // uniform
      quant_unit<T, FMT>(v[j], lane + j * TPR, nchunk, row_ok, row, lane, s_row, bad_row, codes, row_bytes, scales, tiles);
    }
  }
}

// Finite values stay finite: the largest code times a scale rounded up can pass 65504, and nv at the top of bf16's range the largest
// fp32 value too (a row of bf16's largest gets 6 * 352 * 2^117).
__device__ __forceinline__ float clip16(float v, float top) { return v > top ? top : (v < -top ? -top : v); }
__device__ __forceinline__ float finite16(float v, __half) { return clip16(v, 65504.0f); }
__device__ __forceinline__ float finite16(float v, __nv_bfloat16) { return clip16(v, __int_as_float(0x7F7F0000)); }

// A thread turns units of 16 codes (8 bytes and a scale byte) into one 32-byte store each, five units at a time.
template <typename T, int FMT, int TPR>
__global__ void __launch_bounds__(kThreads)
pq_dequant_rows_fp4_kernel(const uint8_t* codes, int64_t ldc, const uint8_t* scales, const float* row_scale, T* out, int64_t ldo,
                           int64_t M, int K) {
  constexpr int RPB = kThreads / TPR;
  T tag{};
  wait_for_previous_kernel();
  const int lane = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
  if (row >= M) return;
  const int nchunk = K >> 4;
  const uint8_t* srow = scales + fp4_scale_off(row, 0, fp4_scale_tiles(K, FMT));
  const float s_row = FMT == PQ_FP4_NV ? row_scale[row] : 1.0f;
  const uint8_t* crow = codes + row * ldc;
  T* orow = out + row * ldo;
  for (int c0 = lane; c0 < nchunk; c0 += kUnits * TPR) {
    uint2 w[kUnits];
    uint32_t byte[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int c = c0 + j * TPR;
      if (c < nchunk) {
        const int blk = FMT == PQ_FP4_MX ? c >> 1 : c;
        w[j] = *reinterpret_cast<const uint2*>(crow + static_cast<int64_t>(c) * 8);
        byte[j] = srow[static_cast<int64_t>(blk >> 2) * 512 + (blk & 3)];      // 2^31 bytes at 2^28 elements (nv)
      }
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int c = c0 + j * TPR;
      if (c >= nchunk) break;
      float s;
      if constexpr (FMT == PQ_FP4_MX)                      // 2^(byte - 127); 2^-127 is subnormal, 255 is NaN
        s = __int_as_float(byte[j] == 255u ? 0x7FC00000 : (byte[j] == 0u ? 0x00400000 : static_cast<int>(byte[j]) << 23));
      else
        s = e4m3_value(byte[j]) * s_row;
      Chunk16 o;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[4];
        unpack_e2m1x8(h == 0 ? w[j].x : w[j].y, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __fmul2_rn(unpack2<__half>(v[i]), make_float2(s, s));
          o.w[4 * h + i] = pack2(finite16(f.x, tag), finite16(f.y, tag), tag);
        }
      }
      st_chunk16(orow + static_cast<int64_t>(c) * 16, o);
    }
  }
}

// The factors of a rank-32 term for the product's accumulator, which stands in units of the row scales.  The first `t_blocks` blocks:
// activations t [M, 32], eight elements per thread, t / s_row in fp32 (exact: a 16-bit value over a power of two).  The others: the
// up-projection B [32, N], transposed, over s_col; a block takes 64 columns, a thread eight elements of one of them, so that a warp
// reads 64 contiguous bytes of a row of B and writes whole 32-byte sectors.  Laying B out costs a fraction of the launch that t needs
// anyway, and nothing has to be kept from call to call: the term is always that of the factor as it is now.
constexpr int kFactorCols = kThreads / 4;
template <typename T, typename TB>
__global__ void __launch_bounds__(kThreads)
pq_fp4_lowrank_factors_kernel(const T* t, const float* row_scale, float* out, int64_t M, unsigned t_blocks, const TB* b, int64_t ldb,
                              const float* col_scale, float* b_out, int64_t N) {
  wait_for_previous_kernel();
  allow_next_kernel();
  if (blockIdx.x >= t_blocks) {
    const int64_t n = static_cast<int64_t>(blockIdx.x - t_blocks) * kFactorCols + threadIdx.x % kFactorCols;
    const int r0 = static_cast<int>(threadIdx.x) / kFactorCols * 8;
    if (n >= N) return;
    const float s = col_scale != nullptr ? col_scale[n] : 1.0f;
    Chunk16 o;
#pragma unroll
    for (int k = 0; k < 8; ++k) o.w[k] = __float_as_uint(__fdiv_rn(static_cast<float>(b[(r0 + k) * ldb + n]), s));
    st_chunk16(b_out + n * 32 + r0, o);
    return;
  }
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= 4 * M) return;
  const float inv = row_scale != nullptr ? 1.0f / row_scale[i >> 2] : 1.0f;
  const uint4 v = *reinterpret_cast<const uint4*>(t + 8 * i);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  T tag{};
  Chunk16 o;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    o.w[2 * k] = __float_as_uint(lo_f32(w[k], tag) * inv);
    o.w[2 * k + 1] = __float_as_uint(hi_f32(w[k], tag) * inv);
  }
  st_chunk16(out + 8 * i, o);
}

struct Args {
  const void* x; int64_t ldx; uint8_t* codes; uint8_t* scales; float* row_scale; int64_t M; int K;
};

template <typename... P, typename... A>
int launch_chained(void (*kern)(P...), int64_t blocks, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at = chained_launch();
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  PQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...));
  return PQ_OK;
}

struct FactorArgs {
  const void* t; const float* row_scale; float* t_out; int64_t M;
  const void* b; int64_t ldb; const float* col_scale; float* b_out; int64_t N;
};
template <typename T, typename TB>
int launch_factors(const FactorArgs& a, cudaStream_t st) {
  const int64_t t_blocks = (4 * a.M + kThreads - 1) / kThreads, blocks = t_blocks + (a.N + kFactorCols - 1) / kFactorCols;
  if (blocks > 0x7fffffffLL) return PQ_ERR_SHAPE;
  return launch_chained(pq_fp4_lowrank_factors_kernel<T, TB>, blocks, st, static_cast<const T*>(a.t), a.row_scale, a.t_out, a.M,
                        static_cast<unsigned>(t_blocks), static_cast<const TB*>(a.b), a.ldb, a.col_scale, a.b_out, a.N);
}

template <typename T, int FMT, int TPR, bool LONG>
int launch_quant(const Args& a, cudaStream_t st) {
  constexpr int RPB = kThreads / TPR;
  const int64_t blocks = (a.M + RPB - 1) / RPB;
  if (blocks > 0x7fffffffLL) return PQ_ERR_SHAPE;
  return launch_chained(pq_quant_rows_fp4_kernel<T, FMT, TPR, LONG>, blocks, st, static_cast<const T*>(a.x), a.ldx, a.codes, a.scales,
                        a.row_scale, a.M, a.K);
}

// the smallest team that keeps the row in registers
template <typename T, int FMT>
int dispatch_quant(const Args& a, cudaStream_t st) {
  const int n = a.K >> 4;
  if (n <= 8 * kUnits) return launch_quant<T, FMT, 8, false>(a, st);
  if (n <= 16 * kUnits) return launch_quant<T, FMT, 16, false>(a, st);
  if (n <= 32 * kUnits) return launch_quant<T, FMT, 32, false>(a, st);
  if (n <= 64 * kUnits) return launch_quant<T, FMT, 64, false>(a, st);
  if (n <= 128 * kUnits) return launch_quant<T, FMT, 128, false>(a, st);
  if (n <= 256 * kUnits) return launch_quant<T, FMT, 256, false>(a, st);
  return launch_quant<T, FMT, 256, true>(a, st);
}

template <typename T, int FMT, int TPR>
int launch_dequant(const void* codes, int64_t ldc, const void* scales, const float* row_scale, void* out, int64_t ldo,
                   int64_t M, int K, cudaStream_t st) {
  constexpr int RPB = kThreads / TPR;
  const int64_t blocks = (M + RPB - 1) / RPB;
  if (blocks > 0x7fffffffLL) return PQ_ERR_SHAPE;
  return launch_chained(pq_dequant_rows_fp4_kernel<T, FMT, TPR>, blocks, st, static_cast<const uint8_t*>(codes), ldc,
                        static_cast<const uint8_t*>(scales), row_scale, static_cast<T*>(out), ldo, M, K);
}
template <typename T, int FMT>
int dispatch_dequant(const void* codes, int64_t ldc, const void* scales, const float* row_scale, void* out, int64_t ldo,
                     int64_t M, int K, cudaStream_t st) {
  const int n = K >> 4;
  if (n <= 8 * kUnits) return launch_dequant<T, FMT, 8>(codes, ldc, scales, row_scale, out, ldo, M, K, st);
  if (n <= 16 * kUnits) return launch_dequant<T, FMT, 16>(codes, ldc, scales, row_scale, out, ldo, M, K, st);
  if (n <= 32 * kUnits) return launch_dequant<T, FMT, 32>(codes, ldc, scales, row_scale, out, ldo, M, K, st);
  return launch_dequant<T, FMT, 64>(codes, ldc, scales, row_scale, out, ldo, M, K, st);
}

}  // namespace
}  // namespace pq

using namespace pq;

extern "C" int64_t pq_fp4_scale_bytes(int64_t M, int64_t K, int fmt) {
  if (M < 0 || K <= 0 || (fmt != PQ_FP4_MX && fmt != PQ_FP4_NV)) return 0;
  return (M + 127) / 128 * fp4_scale_tiles(K, fmt) * 512;
}

extern "C" int pq_quant_rows_fp4(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, int fmt, uint8_t* codes,
                                 uint8_t* scales, float* row_scale, void* stream) {
  if (M < 0 || K <= 0 || K > 0x7fffffffLL || ldx < K) return PQ_ERR_SHAPE;
  if (dtype != PQ_DTYPE_BF16 && dtype != PQ_DTYPE_FP16) return PQ_ERR_DTYPE;
  if (fmt != PQ_FP4_MX && fmt != PQ_FP4_NV) return PQ_ERR_UNSUPPORTED;
  if (M == 0) return PQ_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr || (fmt == PQ_FP4_NV && row_scale == nullptr)) return PQ_ERR_NULL;
  if (K % 32 != 0 || ldx % 16 != 0) return PQ_ERR_ALIGN;
  if (!aligned_to(x, 32) || !aligned_to(codes, 16) || !aligned_to(scales, 16) || !aligned_to(row_scale, 4)) return PQ_ERR_ALIGN;
  const Args a{x, ldx, codes, scales, row_scale, M, static_cast<int>(K)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PQ_DTYPE_BF16)
    return fmt == PQ_FP4_MX ? dispatch_quant<__nv_bfloat16, PQ_FP4_MX>(a, st) : dispatch_quant<__nv_bfloat16, PQ_FP4_NV>(a, st);
  return fmt == PQ_FP4_MX ? dispatch_quant<__half, PQ_FP4_MX>(a, st) : dispatch_quant<__half, PQ_FP4_NV>(a, st);
}

extern "C" int pq_dequant_rows_fp4(const uint8_t* codes, int64_t ldc, const uint8_t* scales, const float* row_scale, int fmt,
                                   void* out, int dtype, int64_t ldo, int64_t M, int64_t K, void* stream) {
  if (M < 0 || K <= 0 || K > 0x7fffffffLL || ldc < K / 2 || ldo < K) return PQ_ERR_SHAPE;
  if (dtype != PQ_DTYPE_BF16 && dtype != PQ_DTYPE_FP16) return PQ_ERR_DTYPE;
  if (fmt != PQ_FP4_MX && fmt != PQ_FP4_NV) return PQ_ERR_UNSUPPORTED;
  if (M == 0) return PQ_OK;
  if (codes == nullptr || scales == nullptr || out == nullptr || (fmt == PQ_FP4_NV && row_scale == nullptr)) return PQ_ERR_NULL;
  if (K % 32 != 0 || ldc % 16 != 0 || ldo % 16 != 0) return PQ_ERR_ALIGN;
  if (!aligned_to(codes, 16) || !aligned_to(scales, 16) || !aligned_to(out, 32) || !aligned_to(row_scale, 4)) return PQ_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PQ_DTYPE_BF16)
    return fmt == PQ_FP4_MX ? dispatch_dequant<__nv_bfloat16, PQ_FP4_MX>(codes, ldc, scales, row_scale, out, ldo, M, static_cast<int>(K), st)
                            : dispatch_dequant<__nv_bfloat16, PQ_FP4_NV>(codes, ldc, scales, row_scale, out, ldo, M, static_cast<int>(K), st);
  return fmt == PQ_FP4_MX ? dispatch_dequant<__half, PQ_FP4_MX>(codes, ldc, scales, row_scale, out, ldo, M, static_cast<int>(K), st)
                          : dispatch_dequant<__half, PQ_FP4_NV>(codes, ldc, scales, row_scale, out, ldo, M, static_cast<int>(K), st);
}

extern "C" int pq_fp4_lowrank_factors(const void* t, int t_dtype, const float* row_scale, float* t_out, int64_t M, const void* b,
                                      int b_dtype, int64_t ldb, const float* col_scale, float* b_out, int64_t N, void* stream) {
  if (M < 0 || N < 0 || M > 0x7fffffffffLL || N > 0x7fffffffffLL || (N > 0 && ldb < N)) return PQ_ERR_SHAPE;
  if ((t_dtype != PQ_DTYPE_BF16 && t_dtype != PQ_DTYPE_FP16) || (b_dtype != PQ_DTYPE_BF16 && b_dtype != PQ_DTYPE_FP16)) return PQ_ERR_DTYPE;
  if (M == 0 && N == 0) return PQ_OK;
  if ((M > 0 && (t == nullptr || t_out == nullptr)) || (N > 0 && (b == nullptr || b_out == nullptr))) return PQ_ERR_NULL;
  if (!aligned_to(t, 16) || !aligned_to(t_out, 32) || !aligned_to(row_scale, 4) || !aligned_to(b, 2) || !aligned_to(b_out, 32) || !aligned_to(col_scale, 4))
    return PQ_ERR_ALIGN;
  const FactorArgs a{t, row_scale, t_out, M, b, ldb, col_scale, b_out, N};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (t_dtype == PQ_DTYPE_BF16)
    return b_dtype == PQ_DTYPE_BF16 ? launch_factors<__nv_bfloat16, __nv_bfloat16>(a, st) : launch_factors<__nv_bfloat16, __half>(a, st);
  return b_dtype == PQ_DTYPE_BF16 ? launch_factors<__half, __nv_bfloat16>(a, st) : launch_factors<__half, __half>(a, st);
}

extern "C" int pq_fp4_lowrank_rows(const void* t, int dtype, const float* row_scale, float* out, int64_t M, void* stream) {
  return pq_fp4_lowrank_factors(t, dtype, row_scale, out, M, nullptr, dtype, 0, nullptr, nullptr, 0, stream);
}
