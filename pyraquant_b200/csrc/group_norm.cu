// Group norm over channels-last rows: z[b,t,c] = act((x[b,t,c] - mean[b,g]) * rstd[b,g] * gamma[c] + beta[c]), statistics over
// the T rows and C / groups channels of a group, act nothing or SiLU (z * sigmoid(z)), one rounding to the 16-bit type.
//
// Two launches.  Both cut the T rows of every sample into P consecutive chunks, one per CTA, and give a thread a fixed
// column of eight channels (one 16-byte load) and every R-th row.
//   1. statistics: a thread sums x - pivot and its square per channel, the pivot being its first value (so that the sum of
//      squares does not cancel when the mean is large against the deviation); means and centred sums of squares of
//      channels, threads and chunks are merged pairwise in a fixed order:
//        n = nA + nB, mean = mA + (mB - mA) nB / n, M2 = M2A + M2B + (mB - mA)^2 nA nB / n.
//   2. the merged statistics of the sample's P chunks, then the normalisation.
// All statistics and arithmetic are fp32.
#include "common.cuh"
#include "quant_common.cuh"

namespace pq {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxC = 8192;
constexpr int kUnroll = 4;

struct NormArgs {
  const void* x; int64_t ld_row, ld_batch;         // elements
  const void* gamma; const void* beta; int affine_f32;
  void* out; int64_t out_row, out_batch;
  float2* part;                                     // [B][P][groups] mean, M2
  int B, T, C, groups, P, silu;
  float eps;
};

struct Stat { float n, mean, m2; };
__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b) {
  Stat r;
  r.n = a.n + b.n;
  const float d = b.mean - a.mean;
  const float w = r.n > 0.0f ? b.n / r.n : 0.0f;
  r.mean = fmaf(d, w, a.mean);
  r.m2 = a.m2 + b.m2 + d * d * a.n * w;
  // an empty side must not bring in what its fields hold
  if (b.n == 0.0f) r = a;
  if (a.n == 0.0f) r = b;
  return r;
}
__device__ __forceinline__ Stat merge_warp(Stat s) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    Stat t;
    t.n = __shfl_down_sync(0xffffffffu, s.n, o);
    t.mean = __shfl_down_sync(0xffffffffu, s.mean, o);
    t.m2 = __shfl_down_sync(0xffffffffu, s.m2, o);
    s = merge(s, t);                                // lane 0 merges lanes 0..31 in order
  }
  return s;
}

// threads over the columns of eight channels: `cols` a pass, R rows side by side
struct Lanes { int ncol, cols, R; };
__host__ __device__ __forceinline__ Lanes lanes_of(int C) {
  Lanes l;
  l.ncol = C >> 3;
  l.cols = l.ncol < kThreads ? l.ncol : kThreads;
  l.R = kThreads / l.cols;
  return l;
}
__host__ __device__ __forceinline__ int chunk_begin(int T, int P, int p) { return static_cast<int>(static_cast<int64_t>(T) * p / P); }

template <typename T>
__global__ void __launch_bounds__(kThreads)
pq_group_norm_stats_kernel(const NormArgs a) {
  extern __shared__ float sm[];                     // [R][C] means, [R][C] M2
  T tag{};
  const Lanes l = lanes_of(a.C);
  const int p = blockIdx.x, b = blockIdx.y;
  const int r0 = chunk_begin(a.T, a.P, p), r1 = chunk_begin(a.T, a.P, p + 1);
  const int rl = static_cast<int>(threadIdx.x) / l.cols;
  const T* xb = static_cast<const T*>(a.x) + static_cast<int64_t>(b) * a.ld_batch;
  float* s_mean = sm;
  float* s_m2 = sm + l.R * a.C;
  if (rl < l.R) {
    for (int col = static_cast<int>(threadIdx.x) % l.cols; col < l.ncol; col += l.cols) {
      float piv[8] = {}, s1[8] = {}, s2[8] = {};
      const T* xc = xb + col * 8;
      int n = 0;
      auto unpack = [&](const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = lo_f32(w[i], tag); f[2 * i + 1] = hi_f32(w[i], tag); }
      };
      if (r0 + rl < r1) {
        float f[8];
        unpack(ld_v4(xc + static_cast<int64_t>(r0 + rl) * a.ld_row), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) piv[i] = f[i];
      }
      for (int r = r0 + rl; r < r1; r += l.R * kUnroll) {
        uint4 v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (r + u * l.R < r1) v[u] = ld_v4(xc + static_cast<int64_t>(r + u * l.R) * a.ld_row);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (r + u * l.R < r1) {
            float f[8];
            unpack(v[u], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) { const float d = f[i] - piv[i]; s1[i] += d; s2[i] = fmaf(d, d, s2[i]); }
            ++n;
          }
      }
      const float inv = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s_mean[rl * a.C + col * 8 + i] = fmaf(s1[i], inv, piv[i]);
        s_m2[rl * a.C + col * 8 + i] = fmaxf(s2[i] - s1[i] * s1[i] * inv, 0.0f);
      }
    }
  }
  __syncthreads();
  const int cpg = a.C / a.groups;
  const int rows = r1 - r0;
  for (int g = static_cast<int>(threadIdx.x) >> 5; g < a.groups; g += kThreads / 32) {
    Stat s{0.0f, 0.0f, 0.0f};
    for (int i = static_cast<int>(threadIdx.x) & 31; i < l.R * cpg; i += 32) {
      const int lane_row = i / cpg, c = g * cpg + i % cpg;
      const int n = rows > lane_row ? (rows - lane_row + l.R - 1) / l.R : 0;
      s = merge(s, Stat{static_cast<float>(n), s_mean[lane_row * a.C + c], s_m2[lane_row * a.C + c]});
    }
    s = merge_warp(s);
    if ((threadIdx.x & 31) == 0) a.part[(static_cast<int64_t>(b) * a.P + p) * a.groups + g] = make_float2(s.mean, s.m2);
  }
}

__device__ __forceinline__ float silu(float z) { return __fdividef(z, 1.0f + __expf(-z)); }

// statistics of the sample's groups from its chunks: s_stat[g] = mean, s_stat[groups + g] = 1 / sqrt(var + eps)
__device__ __forceinline__ void merge_chunks(const NormArgs& a, int b, float* s_stat) {
  const int cpg = a.C / a.groups;
  for (int g = static_cast<int>(threadIdx.x) >> 5; g < a.groups; g += kThreads / 32) {
    Stat s{0.0f, 0.0f, 0.0f};
    for (int p = static_cast<int>(threadIdx.x) & 31; p < a.P; p += 32) {
      const float2 v = a.part[(static_cast<int64_t>(b) * a.P + p) * a.groups + g];
      const float n = static_cast<float>(chunk_begin(a.T, a.P, p + 1) - chunk_begin(a.T, a.P, p)) * static_cast<float>(cpg);
      s = merge(s, Stat{n, v.x, v.y});
    }
    s = merge_warp(s);
    if ((threadIdx.x & 31) == 0) {
      s_stat[g] = s.mean;
      s_stat[a.groups + g] = 1.0f / sqrtf(s.m2 / s.n + a.eps);
    }
  }
}

template <typename T>
__device__ __forceinline__ float affine_at(const void* v, int c, int f32, float none) {
  if (v == nullptr) return none;
  if (f32) return static_cast<const float*>(v)[c];
  return lo_f32(static_cast<const unsigned short*>(v)[c], T{});
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
pq_group_norm_apply_kernel(const NormArgs a) {
  extern __shared__ float sm[];                     // [2][groups]
  T tag{};
  const Lanes l = lanes_of(a.C);
  const int p = blockIdx.x, b = blockIdx.y;
  const int r0 = chunk_begin(a.T, a.P, p), r1 = chunk_begin(a.T, a.P, p + 1);
  merge_chunks(a, b, sm);
  __syncthreads();
  const int rl = static_cast<int>(threadIdx.x) / l.cols;
  if (rl >= l.R) return;
  const int cpg = a.C / a.groups;
  for (int col = static_cast<int>(threadIdx.x) % l.cols; col < l.ncol; col += l.cols) {
    float mean[8], mul[8], add[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col * 8 + i, g = c / cpg;
      mean[i] = sm[g];
      mul[i] = sm[a.groups + g] * affine_at<T>(a.gamma, c, a.affine_f32, 1.0f);
      add[i] = affine_at<T>(a.beta, c, a.affine_f32, 0.0f);
    }
    const T* xc = static_cast<const T*>(a.x) + static_cast<int64_t>(b) * a.ld_batch + col * 8;
    T* oc = static_cast<T*>(a.out) + static_cast<int64_t>(b) * a.out_batch + col * 8;
    for (int r = r0 + rl; r < r1; r += l.R * kUnroll) {
      uint4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (r + u * l.R < r1) v[u] = ld_v4(xc + static_cast<int64_t>(r + u * l.R) * a.ld_row);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (r + u * l.R < r1) {
          const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float z0 = fmaf(lo_f32(w[i], tag) - mean[2 * i], mul[2 * i], add[2 * i]);
            float z1 = fmaf(hi_f32(w[i], tag) - mean[2 * i + 1], mul[2 * i + 1], add[2 * i + 1]);
            if (a.silu) { z0 = silu(z0); z1 = silu(z1); }
            o[i] = pack2(z0, z1, tag);
          }
          st_v4(oc + static_cast<int64_t>(r + u * l.R) * a.out_row, make_uint4(o[0], o[1], o[2], o[3]));
        }
    }
  }
}

// chunks per sample: all SMs busy, at least one unrolled step of rows per CTA
int chunks_of(int B, int T, int C) {
  const Lanes l = lanes_of(C);
  int P = 2 * sm_count() / B;
  const int most = (T + l.R * kUnroll - 1) / (l.R * kUnroll);
  if (P > most) P = most;
  return P < 1 ? 1 : P;
}

template <typename T>
int launch_norm(const NormArgs& a, cudaStream_t st) {
  const Lanes l = lanes_of(a.C);
  const dim3 grid(static_cast<unsigned>(a.P), static_cast<unsigned>(a.B));
  const int smem = 2 * l.R * a.C * static_cast<int>(sizeof(float));
  if (smem > 48 * 1024)
    PQ_CUDA_TRY(cudaFuncSetAttribute(pq_group_norm_stats_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  pq_group_norm_stats_kernel<T><<<grid, kThreads, smem, st>>>(a);
  PQ_CUDA_TRY(cudaGetLastError());
  pq_group_norm_apply_kernel<T><<<grid, kThreads, 2 * a.groups * static_cast<int>(sizeof(float)), st>>>(a);
  PQ_CUDA_TRY(cudaGetLastError());
  return PQ_OK;
}

}  // namespace
}  // namespace pq

using namespace pq;

extern "C" int64_t pq_group_norm_workspace_bytes(int64_t B, int64_t T, int64_t C, int groups) {
  if (B <= 0 || T <= 0 || C <= 0 || groups <= 0 || B > 65535 || T > 0x7fffffffLL || C > kMaxC) return 0;
  return B * chunks_of(static_cast<int>(B), static_cast<int>(T), static_cast<int>(C)) * groups * static_cast<int64_t>(sizeof(float2));
}

extern "C" int pq_group_norm(const void* x, int dtype, int64_t B, int64_t T, int64_t C, int64_t ld_row, int64_t ld_batch,
                             int groups, const void* gamma, const void* beta, int affine_fp32, float eps, int act,
                             void* out, int64_t ldo_row, int64_t ldo_batch, void* workspace, int64_t ws_bytes, void* stream) {
  if (B < 0 || T < 0 || C <= 0 || groups <= 0 || B > 65535 || T > 0x7fffffffLL || C > kMaxC || C % groups != 0) return PQ_ERR_SHAPE;
  if (!(eps >= 0.0f) || ld_row < C || ldo_row < C || ld_batch < 0 || ldo_batch < 0) return PQ_ERR_SHAPE;
  if (dtype != PQ_DTYPE_BF16 && dtype != PQ_DTYPE_FP16) return PQ_ERR_DTYPE;
  if (act != PQ_ACT_NONE && act != PQ_ACT_SILU) return PQ_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return PQ_OK;
  if (x == nullptr || out == nullptr || workspace == nullptr) return PQ_ERR_NULL;
  if (C % 8 != 0 || ld_row % 8 != 0 || ld_batch % 8 != 0 || ldo_row % 8 != 0 || ldo_batch % 8 != 0) return PQ_ERR_ALIGN;
  if (!aligned_to(x, 16) || !aligned_to(out, 16) || !aligned_to(workspace, 8) || !aligned_to(gamma, affine_fp32 ? 4 : 2) ||
      !aligned_to(beta, affine_fp32 ? 4 : 2))
    return PQ_ERR_ALIGN;
  if (ws_bytes < pq_group_norm_workspace_bytes(B, T, C, groups)) return PQ_ERR_WORKSPACE;
  NormArgs a{};
  a.x = x; a.ld_row = ld_row; a.ld_batch = ld_batch; a.gamma = gamma; a.beta = beta; a.affine_f32 = affine_fp32 != 0;
  a.out = out; a.out_row = ldo_row; a.out_batch = ldo_batch; a.part = static_cast<float2*>(workspace);
  a.B = static_cast<int>(B); a.T = static_cast<int>(T); a.C = static_cast<int>(C); a.groups = groups;
  a.P = chunks_of(a.B, a.T, a.C); a.silu = act == PQ_ACT_SILU; a.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == PQ_DTYPE_BF16 ? launch_norm<__nv_bfloat16>(a, st) : launch_norm<__half>(a, st);
}
