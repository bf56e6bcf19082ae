// Group norm over channels-last rows: z[b,t,c] = act((x[b,t,c] - mean[b,g]) * rstd[b,g] * gamma[c] + beta[c]), statistics over
// the T rows and C / groups channels of a group, act nothing or SiLU (z * sigmoid(z)), one rounding to the 16-bit type;
// with or without the per-row quantisation of z (INT8, mx, nv) in the same launch.
//
// Cannot do without 2 bytes read and 2 (z), 1 (INT8) or 0.53 to 0.56 (4-bit) written per element, provided x is read once although
// the statistics are needed before the first output.  What bounds it while the rows fit on the chip is latency: 5 of 16 us between
// the sweeps, then chains of dependent operations (4 x 16384 x 320: issue slots 49 % used, no pipe above 31 %); beyond that HBM, with
// the second reading.  One cooperative launch of one CTA per SM: the T rows of a sample are
// cut into P consecutive chunks, one per CTA, which pass through a ring of four segments in shared memory (200 KB, 30 MB
// over the GPU) by bulk copies, and what the ring holds at the end of the first pass is not read again for the second.
//   1. First to last segment: a thread has a fixed column of eight channels and every R-th row and sums x - pivot and its
//      square per channel, the pivot being its first value (the sum of squares must not cancel when the mean is large
//      against the deviation).  The CTA's mean of a group is the sum of the threads' sums, its centred sum of squares that
//      of M2_thread + n (mean_thread - mean)^2: no cancellation, fixed order.
//   2. After a grid barrier every CTA does the same with the P chunks of its sample, and normalises its rows, last to
//      first segment: the last four are there, of the others the ones read last are the likeliest to be in L2 still.
// The quantising forms put z back into shared memory, take every row's largest magnitude (an atomic maximum of bit patterns,
// independent of order) and write codes in a third sweep; they need all rows of a chunk in the ring.
// All statistics and arithmetic are fp32.
#include <cooperative_groups.h>

#include "common.cuh"
#include "fp4_common.cuh"
#include "quant_common.cuh"

namespace pq {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxC = 8192;
constexpr int kSlots = 4;                         // segments in shared memory (1 x 262144 x 256: eight 75.5 us, four 73.6)
constexpr int kSmemMax = 232448;
// steps of R rows that one CTA takes alone, without cooperative launch and barrier: us, shared / alone, 12 x 640 (two steps)
// 7.2 / 5.7, 18 x 640 (three) 7.2 / 6.3 and with nv codes 8.2 / 7.9; every further step adds 0.5
constexpr int kAloneSteps = 3;
constexpr int kPartsPerLane = 5;                  // chunks of a sample: at most 160

enum Mode { kOut16 = 0, kInt8 = 1, kMx = 2, kNv = 3 };

// threads over the columns of eight channels: `cols` a pass, R rows side by side
struct Lanes { int ncol, cols, R; };
__host__ __device__ __forceinline__ Lanes lanes_of(int C) {
  Lanes l;
  l.ncol = C >> 3;
  l.cols = l.ncol < kThreads ? l.ncol : kThreads;
  l.R = kThreads / l.cols;
  return l;
}

// shared memory: ring of rows, then per-thread sums [R][C], group statistics [2][groups], row maxima (quantising forms, whose rows
// all fit), barriers full[kSlots], empty[kSlots]
struct NormSmem {
  int red, stat, amax, bars, total;
};
__host__ __device__ __forceinline__ NormSmem smem_of(int C, int groups, int ring_rows) {
  NormSmem s;
  s.red = (ring_rows * C * 2 + 127) & ~127;
  s.stat = s.red + lanes_of(C).R * C * 4;
  s.amax = s.stat + 2 * groups * 4;
  s.bars = (s.amax + ring_rows * 4 + 7) & ~7;
  s.total = s.bars + 2 * kSlots * 8;
  return s;
}

struct NormArgs {
  const void* x; int64_t ld_row, ld_batch;         // elements
  const void* gamma; const void* beta; int affine_f32;
  void* out; int64_t out_row, out_batch;            // z (NULL: not wanted)
  uint8_t* codes;                                   // INT8 [B T, C] or packed E2M1 [B T, C / 2]
  uint8_t* scales;                                  // 4-bit: scale tiles
  float* row_scale;                                 // INT8, nv
  float2* part;                                     // [B][groups][P] mean, M2
  int32_t* status;
  int B, T, C, groups, P, silu;
  int seg_rows;                                     // rows of a segment
  int chunk, longer;                                // rows per chunk; the first `longer` chunks have one more
  // what follows from the sizes, worked out on the host: a division on the way to the first copy costs a tenth of a
  // microsecond, and there would be eight of them
  Lanes l; NormSmem lay;
  int cpg, nch, R2;                                 // channels per group; units of 16 channels, rows of them side by side
  float inv_cpg, inv_cols, inv_nch, inv_R;
  float eps;
};

// c / cpg for 0 <= c < 8192: (c + 1/2) / cpg is at least 1 / (2 cpg) away from an integer and its rounding error below
// c / cpg * 2^-22, which is less as long as C < 2^21
__device__ __forceinline__ int group_of(int c, float inv_cpg) { return static_cast<int>((static_cast<float>(c) + 0.5f) * inv_cpg); }

__device__ __forceinline__ float ex2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// the larger of the two, NaN if one of them is
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// z * sigmoid(z) = z / (1 + 2^t), t = -z log2(e), for two values with one reciprocal: 1 / d0 = d1 / (d0 d1).  An exponential and a
// reciprocal per value would keep the special-function pipe busy for 16 cycles a warp; this takes 12, next to about ten
// instructions a value in all.  t is held at 60 so that the product stays finite and a NaN leaves its partner alone; the sigmoid then
// ends at 2^-60, and the z beside it is held at -41.6 (t = 60.02): from there down the function lies between -4e-17 and 0 and comes out
// as -41.6 * 2^-60 = -3.6e-17 however far down z is.  us without / with that hold: 1 x 1024 x 1280 9.0 / 9.1, 2 x 16384 x 320 15.5 /
// 16.0, 1 x 262144 x 256 74.0 / 75.2; a select that ends at zero, or one test for several values, costs a little more.
__device__ __forceinline__ float2 silu2(float2 z) {
  const float2 t = __fmul2_rn(z, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 e = make_float2(ex2_approx(fminf(t.x, 60.0f)), ex2_approx(fminf(t.y, 60.0f)));
  const float2 d = __fadd2_rn(e, make_float2(1.0f, 1.0f));
  const float r = rcp_approx(d.x * d.y);
  return __fmul2_rn(make_float2(max_or_nan(z.x, -41.6f), max_or_nan(z.y, -41.6f)), make_float2(r * d.y, r * d.x));
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float2 (&f)[4]) {
  f[0] = unpack2<T>(v.x); f[1] = unpack2<T>(v.y); f[2] = unpack2<T>(v.z); f[3] = unpack2<T>(v.w);
}
// contiguous copy global -> shared, completion bytes on a barrier of this CTA; 16-byte aligned, size % 16 == 0
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// running sums of one column of eight channels; after finish(): means in neg (negated), centred sums of squares in s2
struct ColumnSums {
  float2 neg[4], s1[4], s2[4];          // -pivot, sum of x - pivot, of its square
  float count;
  __device__ __forceinline__ float mean(int i) const { return -(i & 1 ? neg[i >> 1].y : neg[i >> 1].x); }
  __device__ __forceinline__ float m2(int i) const { return i & 1 ? s2[i >> 1].y : s2[i >> 1].x; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) neg[i] = s1[i] = s2[i] = make_float2(0.0f, 0.0f);
  }
  template <typename T>
  __device__ __forceinline__ void pivot(const uint4& v) {
    float2 f[4];
    unpack8<T>(v, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) neg[i] = make_float2(-f[i].x, -f[i].y);
  }
  template <typename T>
  __device__ __forceinline__ void add(const uint4& v) {
    float2 f[4];
    unpack8<T>(v, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = __fadd2_rn(f[i], neg[i]);
      s1[i] = __fadd2_rn(s1[i], d);
      s2[i] = __ffma2_rn(d, d, s2[i]);
    }
  }
  __device__ __forceinline__ void finish(int n) {
    count = static_cast<float>(n);
    const float inv = n > 0 ? 1.0f / count : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s2[i] = make_float2(fmaxf(s2[i].x - s1[i].x * s1[i].x * inv, 0.0f), fmaxf(s2[i].y - s1[i].y * s1[i].y * inv, 0.0f));
      neg[i] = make_float2(fmaf(-s1[i].x, inv, neg[i].x), fmaf(-s1[i].y, inv, neg[i].y));
    }
  }
};

template <typename F>
__device__ __forceinline__ void put8(float* dst, F&& f) {
  *reinterpret_cast<float4*>(dst) = make_float4(f(0), f(1), f(2), f(3));
  *reinterpret_cast<float4*>(dst + 4) = make_float4(f(4), f(5), f(6), f(7));
}

// The normalisation of eight channels: gamma and beta are requested before the grid barrier (and left as they were loaded:
// converting them would wait for them), the statistics come after it.
template <typename T>
struct Affine8 {
  uint4 raw[2][2];                        // gamma, beta: eight 16-bit values in [0], or eight fp32 ones
  float2 mul[4], add[4];                  // z = x mul + add; add holds -mean mul too, which costs half a unit of 2^-24 |mean| / std
  __device__ __forceinline__ void request(const NormArgs& a, int c0) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const void* v = k == 0 ? a.gamma : a.beta;
      if (v == nullptr) continue;
      if (a.affine_f32) {
        raw[k][0] = ld_v4(static_cast<const float*>(v) + c0);
        raw[k][1] = ld_v4(static_cast<const float*>(v) + c0 + 4);
      } else {
        raw[k][0] = ld_v4(static_cast<const T*>(v) + c0);
      }
    }
  }
  __device__ __forceinline__ void values(const NormArgs& a, int k, float none, float2 (&o)[4]) const {
    if ((k == 0 ? a.gamma : a.beta) == nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = make_float2(none, none);
    } else if (a.affine_f32) {
      const uint4 u = raw[k][0], w = raw[k][1];
      o[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y)); o[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
      o[2] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y)); o[3] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    } else {
      unpack8<T>(raw[k][0], o);
    }
  }
  __device__ __forceinline__ void complete(const NormArgs& a, const float* stat, int c0) {
    values(a, 0, 1.0f, mul);
    values(a, 1, 0.0f, add);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g0 = group_of(c0 + 2 * i, a.inv_cpg), g1 = group_of(c0 + 2 * i + 1, a.inv_cpg);
      mul[i] = __fmul2_rn(mul[i], make_float2(stat[a.groups + g0], stat[a.groups + g1]));
      add[i] = __ffma2_rn(make_float2(-stat[g0], -stat[g1]), mul[i], add[i]);
    }
  }
  __device__ __forceinline__ void both(const uint4& v, const uint4& w, int with_silu, uint4& zv, uint4& zw) const {
    float2 f[4], g[4];
    unpack8<T>(v, f);
    unpack8<T>(w, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __ffma2_rn(f[i], mul[i], add[i]);
      g[i] = __ffma2_rn(g[i], mul[i], add[i]);
    }
    if (with_silu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[i] = silu2(f[i]); g[i] = silu2(g[i]); }
    }
    T tag{};
    zv = make_uint4(pack2(f[0].x, f[0].y, tag), pack2(f[1].x, f[1].y, tag), pack2(f[2].x, f[2].y, tag), pack2(f[3].x, f[3].y, tag));
    zw = make_uint4(pack2(g[0].x, g[0].y, tag), pack2(g[1].x, g[1].y, tag), pack2(g[2].x, g[2].y, tag), pack2(g[3].x, g[3].y, tag));
  }
  __device__ __forceinline__ uint4 operator()(const uint4& v, int with_silu) const {
    float2 f[4];
    unpack8<T>(v, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __ffma2_rn(f[i], mul[i], add[i]);
    if (with_silu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = silu2(f[i]);
    }
    T tag{};
    return make_uint4(pack2(f[0].x, f[0].y, tag), pack2(f[1].x, f[1].y, tag), pack2(f[2].x, f[2].y, tag), pack2(f[3].x, f[3].y, tag));
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums over the R x cpg entries of every group of `red`, in a fixed order; a warp for two groups at a time in the usual case of at
// most 128 entries (32 groups whose columns nearly fill the threads), whose places are worked out once.
struct GroupSums {
  int off[4], R, C, groups, cpg;
  __device__ __forceinline__ void init(const NormArgs& a) {
    R = a.l.R; C = a.C; groups = a.groups; cpg = a.cpg;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = lane + 32 * k, r = group_of(i, a.inv_cpg);
      off[k] = i < R * cpg ? r * C + i - r * cpg : -1;
    }
  }
  template <typename F>
  __device__ __forceinline__ void operator()(const float* red, F&& put) const {
    const int lane = threadIdx.x & 31;
    if (R * cpg <= 128) {
      for (int g = static_cast<int>(threadIdx.x) >> 5; g < groups; g += 2 * kWarps) {
        const int h = g + kWarps;
        const float* rg = red + g * cpg;
        const float* rh = red + h * cpg;
        float s = 0.0f, t = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (off[k] >= 0) s += rg[off[k]];
          if (off[k] >= 0 && h < groups) t += rh[off[k]];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); t += __shfl_xor_sync(0xffffffffu, t, o); }
        if (lane == 0) put(g, s);
        if (lane == 1 && h < groups) put(h, t);
      }
    } else {
#pragma unroll 1
      for (int g = static_cast<int>(threadIdx.x) >> 5; g < groups; g += kWarps) {
        float s = 0.0f;
        if (cpg >= 32) {
#pragma unroll 1
          for (int r = 0; r < R; ++r)
            for (int c = lane; c < cpg; c += 32) s += red[r * C + g * cpg + c];
        } else {
          const int per = 32 / cpg, r0 = lane / cpg, c = lane - r0 * cpg;      // floor(32 / cpg) rows at a time
          if (r0 < per)
            for (int r = r0; r < R; r += per) s += red[r * C + g * cpg + c];
        }
        s = warp_sum(s);
        if (lane == 0) put(g, s);
      }
    }
  }
};

// COLS: columns of eight channels per thread, two only for C > 4096
template <typename T, int MODE, int COLS>
__global__ void __launch_bounds__(kThreads, 1)
pq_group_norm_kernel(const NormArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  if constexpr (MODE != kOut16) allow_next_kernel();                     // the product that takes these rows
  T tag{};
  const Lanes l = a.l;
  const NormSmem lay = a.lay;
  float* red = reinterpret_cast<float*>(smem + lay.red);
  float* stat = reinterpret_cast<float*>(smem + lay.stat);              // mean, then 1 / sqrt(var + eps)
  uint32_t* amax = reinterpret_cast<uint32_t*>(smem + lay.amax);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + lay.bars);
  const uint32_t rows_s = smem_u32(smem);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int p = static_cast<int>(blockIdx.x);
  const int r0 = p * a.chunk + (p < a.longer ? p : a.longer), rows = a.chunk + (p < a.longer ? 1 : 0);
  const int segs = (rows + a.seg_rows - 1) / a.seg_rows;
  const int cpg = a.cpg;
  const float inv_cpg = a.inv_cpg;
  const int rl = group_of(tid, a.inv_cols), col0 = tid - rl * l.cols;
  const int row_bytes = a.C * 2, slot_bytes = a.seg_rows * row_bytes;
  uint64_t* empty = bars + kSlots;

#pragma unroll 1
  for (int b = static_cast<int>(blockIdx.y); b < a.B; b += static_cast<int>(gridDim.y)) {
    const T* xb = static_cast<const T*>(a.x) + static_cast<int64_t>(b) * a.ld_batch + static_cast<int64_t>(r0) * a.ld_row;
    // segment s into its slot; one lane for contiguous rows, the lanes of a warp side by side for others
    auto load = [&](int s) {
      const int from = s * a.seg_rows, n = min(a.seg_rows, rows - from);
      const uint32_t dst = rows_s + (s % kSlots) * slot_bytes;
      uint64_t* bar = &bars[s % kSlots];
      if (a.ld_row == a.C) {
        mbar_arrive_expect_tx(bar, static_cast<uint32_t>(n * row_bytes));
        bulk_copy(dst, xb + static_cast<int64_t>(from) * a.C, static_cast<uint32_t>(n * row_bytes), bar);
      } else {
        if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(n * row_bytes));
        __syncwarp();
        for (int r = lane; r < n; r += 32)
          bulk_copy(dst + r * row_bytes, xb + static_cast<int64_t>(from + r) * a.ld_row, static_cast<uint32_t>(row_bytes), bar);
      }
    };
    // In both passes the segment's wait has the parity of s / kSlots: the first pass fills a slot L + 1 times, with its segments
    // 0 .. L, the second refills it with L - 1 .. 0, fill number 2 L - q for segment q.  The slot is given back once per
    // segment and pass, 2 L + 1 - q times before by segment q of the second pass.
    auto wait_full = [&](int s) {
      if (!mbar_wait_bounded(&bars[s % kSlots], (s / kSlots) & 1)) report_timeout(a.status, 8, 1);
    };
    auto refill = [&](int used, int s, uint32_t parity) {             // warp 0: segment s once everybody is done with `used`
      if (a.ld_row != a.C || lane == 0) {
        if (!mbar_wait_bounded(&empty[used % kSlots], parity)) report_timeout(a.status, 8, 2);
        load(s);
      }
      __syncwarp();
    };
    // ---------------------------------------------------------------- the first segments on their way
    if (warp == 0) {
      if (lane < kSlots) {
        if (b != static_cast<int>(blockIdx.y)) {                      // another sample: barriers from the start
          asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(smem_u32(&bars[lane])) : "memory");
          asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(smem_u32(&empty[lane])) : "memory");
        }
        mbar_init(&bars[lane], 1);
        mbar_init(&empty[lane], kWarps);
        fence_mbar_init();
        fence_proxy_async_smem();
        if (a.ld_row == a.C && lane < segs) load(lane);
      }
      __syncwarp();
      if (a.ld_row != a.C)
        for (int s = 0; s < min(segs, kSlots); ++s) load(s);
    }
    if (MODE != kOut16)
      for (int r = tid; r < rows; r += kThreads) amax[r] = 0u;
    GroupSums group_sums;
    group_sums.init(a);
    const float inv_count = 1.0f / (static_cast<float>(rows) * static_cast<float>(cpg));
    __syncthreads();                                                     // barriers and row maxima are there

    // ---------------------------------------------------------------- statistics of the chunk
    ColumnSums cs[COLS];
#pragma unroll
    for (int k = 0; k < COLS; ++k) cs[k].clear();
    int taken = 0;
#pragma unroll 1
    for (int s = 0; s < segs; ++s) {
      wait_full(s);
      const int n = min(a.seg_rows, rows - s * a.seg_rows);
      const uint32_t at = rows_s + (s % kSlots) * slot_bytes + col0 * 16;
#pragma unroll
      for (int k = 0; k < COLS; ++k)
        if (rl < l.R && col0 + k * l.cols < l.ncol) {
          if (taken == 0 && rl < n) cs[k].template pivot<T>(ld_shared_v4(at + rl * row_bytes + k * l.cols * 16));
#pragma unroll 2
          for (int r = rl; r < n; r += l.R) cs[k].template add<T>(ld_shared_v4(at + r * row_bytes + k * l.cols * 16));
        }
      if (rl < n) taken += group_of(n - rl + l.R - 1, a.inv_R);           // rows this thread has taken
      if (segs > kSlots) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s % kSlots]);
        if (warp == 0 && s >= 1 && s - 1 + kSlots < segs) refill(s - 1, s - 1 + kSlots, ((s - 1) / kSlots) & 1);
      }
    }
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      cs[k].finish(taken);
      const int col = col0 + k * l.cols;
      if (rl < l.R && col < l.ncol) put8(red + rl * a.C + col * 8, [&](int i) { return cs[k].mean(i) * cs[k].count; });
    }
    __syncthreads();
    group_sums(red, [&](int g, float s) { stat[g] = s * inv_count; });
    __syncthreads();
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      const int col = col0 + k * l.cols;
      if (rl < l.R && col < l.ncol)
        put8(red + rl * a.C + col * 8, [&](int i) {
          const float d = cs[k].mean(i) - stat[group_of(col * 8 + i, inv_cpg)];
          return fmaf(d * d, cs[k].count, cs[k].m2(i));
        });
    }
    __syncthreads();
    group_sums(red, [&](int g, float s) { stat[a.groups + g] = s; });
    __syncthreads();

    Affine8<T> f;
    if (rl < l.R) f.request(a, col0 * 8);

    // ---------------------------------------------------------------- statistics of the sample
    if (a.P > 1) {
      for (int g = tid; g < a.groups; g += kThreads)
        a.part[(static_cast<int64_t>(b) * a.groups + g) * a.P + p] = make_float2(stat[g], stat[a.groups + g]);
      cooperative_groups::this_grid().sync();
      const float inv_total = 1.0f / (static_cast<float>(a.T) * static_cast<float>(cpg));
      const float n_long = static_cast<float>((a.chunk + 1) * cpg), n_short = static_cast<float>(a.chunk * cpg);
      // a warp for two groups at a time: their loads are in flight together
#pragma unroll 1
      for (int g = warp; g < a.groups; g += 2 * kWarps) {
        const int h = g + kWarps < a.groups ? g + kWarps : g;
        const float2* part_g = a.part + (static_cast<int64_t>(b) * a.groups + g) * a.P;
        const float2* part_h = a.part + (static_cast<int64_t>(b) * a.groups + h) * a.P;
        float2 u[kPartsPerLane], v[kPartsPerLane];
#pragma unroll
        for (int k = 0; k < kPartsPerLane; ++k) {
          const int i = lane + 32 * k;
          u[k] = i < a.P ? __ldcg(part_g + i) : make_float2(0.0f, 0.0f);
          v[k] = i < a.P ? __ldcg(part_h + i) : make_float2(0.0f, 0.0f);
        }
        float n[kPartsPerLane], su = 0.0f, sv = 0.0f;
#pragma unroll
        for (int k = 0; k < kPartsPerLane; ++k) {
          const int i = lane + 32 * k;
          n[k] = i < a.longer ? n_long : (i < a.P ? n_short : 0.0f);
          su = fmaf(u[k].x, n[k], su); sv = fmaf(v[k].x, n[k], sv);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { su += __shfl_xor_sync(0xffffffffu, su, o); sv += __shfl_xor_sync(0xffffffffu, sv, o); }
        const float mean_u = su * inv_total, mean_v = sv * inv_total;
        su = sv = 0.0f;
#pragma unroll
        for (int k = 0; k < kPartsPerLane; ++k) {
          const float du = u[k].x - mean_u, dv = v[k].x - mean_v;
          su += fmaf(du * du, n[k], u[k].y); sv += fmaf(dv * dv, n[k], v[k].y);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { su += __shfl_xor_sync(0xffffffffu, su, o); sv += __shfl_xor_sync(0xffffffffu, sv, o); }
        if (lane == 0) { stat[g] = mean_u; stat[a.groups + g] = 1.0f / sqrtf(su * inv_total + a.eps); }
        if (lane == 1) { stat[h] = mean_v; stat[a.groups + h] = 1.0f / sqrtf(sv * inv_total + a.eps); }
      }
    } else {
      for (int g = tid; g < a.groups; g += kThreads) stat[a.groups + g] = 1.0f / sqrtf(stat[a.groups + g] * inv_count + a.eps);
    }
    __syncthreads();

    // ---------------------------------------------------------------- normalisation
    const int64_t out0 = static_cast<int64_t>(b) * a.out_batch + static_cast<int64_t>(r0) * a.out_row;
    if constexpr (MODE == kOut16) {
      const bool ring = segs > kSlots;                                    // else one sweep over rows that are all there
#pragma unroll 1
      for (int s = ring ? segs - 1 : 0; s >= 0; --s) {
        if (s < segs - kSlots) wait_full(s);
        const int n = ring ? min(a.seg_rows, rows - s * a.seg_rows) : rows;
        const uint32_t at = rows_s + (s % kSlots) * slot_bytes;
#pragma unroll 1
        for (int k = 0; k < COLS; ++k) {
          const int col = col0 + k * l.cols;
          if (rl >= l.R || col >= l.ncol) break;
          if (COLS > 1) f.request(a, col * 8);
          if (COLS > 1 || !ring || s == segs - 1) f.complete(a, stat, col * 8);
          T* oc = static_cast<T*>(a.out) + out0 + static_cast<int64_t>(s * a.seg_rows) * a.out_row + col * 8;
          // two rows at a time: their chains of dependent operations interleave
          int r = rl;
#pragma unroll 1
          for (; r + l.R < n; r += 2 * l.R) {
            const uint4 v0 = ld_shared_v4(at + r * row_bytes + col * 16), v1 = ld_shared_v4(at + (r + l.R) * row_bytes + col * 16);
            uint4 z0, z1;
            f.both(v0, v1, a.silu, z0, z1);
            st_v4_cs(oc + static_cast<int64_t>(r) * a.out_row, z0);
            st_v4_cs(oc + static_cast<int64_t>(r + l.R) * a.out_row, z1);
          }
          if (r < n) st_v4_cs(oc + static_cast<int64_t>(r) * a.out_row, f(ld_shared_v4(at + r * row_bytes + col * 16), a.silu));
        }
        if (ring) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[s % kSlots]);
          // the segment done before this one makes room; its slot's next one, going down, is kSlots before it
          if (warp == 0 && s + 1 < segs && s + 1 - kSlots >= 0) refill(s + 1, s + 1 - kSlots, (((s + 1) / kSlots) & 1) ^ 1u);
        }
      }
    } else {
      // lanes of one row that share an atomic maximum: eight, four, two or one neighbours, as the columns divide
      const int share = (l.ncol & 7) == 0 ? 8 : ((l.ncol & 3) == 0 ? 4 : ((l.ncol & 1) == 0 ? 2 : 1));
#pragma unroll 1
      for (int k = 0; k < COLS; ++k) {
        const int col = col0 + k * l.cols;
        const bool mine = rl < l.R && col < l.ncol;
        if (mine) {
          if (COLS > 1) f.request(a, col * 8);
          f.complete(a, stat, col * 8);
        }
#pragma unroll 2
        for (int rb = 0; rb < rows; rb += l.R) {
          const int r = rb + rl;
          const bool ok = mine && r < rows;
          uint32_t m = 0u;
          if (ok) {
            const uint32_t at = rows_s + r * row_bytes + col * 16;
            const uint4 z = f(ld_shared_v4(at), a.silu);
            st_shared_v4(at, z);
            if (a.out != nullptr) st_v4_cs(static_cast<T*>(a.out) + out0 + static_cast<int64_t>(r) * a.out_row + col * 8, z);
            if constexpr (MODE != kMx) m = max_pattern(absmax_chunk<T>(0u, z));
          }
          if constexpr (MODE != kMx) {
            if (share >= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            if (share >= 4) m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            if (share >= 8) m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
            if (ok && (tid & (share - 1)) == 0) atomicMax(&amax[r], m);
          }
        }
      }
    }
    if constexpr (MODE != kOut16) {
      __syncthreads();
      // a thread has a fixed column of 16 channels and every R2-th row
      const int nch = a.nch, R2 = a.R2;
      const int r2 = group_of(tid, a.inv_nch), ci = tid - r2 * nch;
      const bool active = r2 < R2;
      const int64_t tiles = MODE == kInt8 ? 0 : fp4_scale_tiles(a.C, MODE == kMx ? PQ_FP4_MX : PQ_FP4_NV);
#pragma unroll 1
      for (int rb = 0; rb < rows; rb += R2) {
        const int r = rb + r2;
        const bool ok = active && r < rows;
        const int64_t row = static_cast<int64_t>(b) * a.T + r0 + r;
        uint4 z0 = make_uint4(0u, 0u, 0u, 0u), z1 = z0;
        if (ok) {
          const uint32_t at = rows_s + r * row_bytes + ci * 32;
          z0 = ld_shared_v4(at); z1 = ld_shared_v4(at + 16);
        }
        if constexpr (MODE == kInt8) {
          if (!ok) continue;
          const QuantScale qs = make_quant_scale(lo_f32(amax[r], tag));
          if (ci == 0) a.row_scale[row] = qs.scale;
          uint4 q;
          quant_chunk<T>(z0, qs, q.x, q.y);
          quant_chunk<T>(z1, qs, q.z, q.w);
          st_v4(a.codes + row * a.C + ci * 16, q);
        } else {
          const Chunk16 c{{z0.x, z0.y, z0.z, z0.w, z1.x, z1.y, z1.z, z1.w}};
          uint32_t m = max_pattern(absmax_chunk16(c));
          BlockScale s;
          if constexpr (MODE == kMx) {
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));               // C % 32 == 0: a block is two neighbours
            s = mx_block_scale(lo_f32(m, tag));
          } else {
            const float top = ok ? lo_f32(amax[r], tag) : 0.0f;
            const bool bad = (__float_as_int(top) >> 23) == 255;
            const float s_row = bad ? 1.0f : nv_row_scale(top);
            s = nv_block_scale(lo_f32(m, tag), s_row, bad);
            if (ok && ci == 0) a.row_scale[row] = bad ? __int_as_float(0x7FC00000) : s_row;
          }
          if (!ok) continue;
          const uint2 q = quant_chunk16<T, MODE == kMx ? PQ_FP4_MX : PQ_FP4_NV>(c, s);
          st_v2(a.codes + row * (a.C >> 1) + ci * 8, q.x, q.y);
          const int blk = MODE == kMx ? ci >> 1 : ci, blocks = MODE == kMx ? nch >> 1 : nch;
          if (MODE == kNv || (ci & 1) == 0) {
            uint8_t* sp = a.scales + fp4_scale_off(row, blk >> 2, tiles) + (blk & 3);
            *sp = static_cast<uint8_t>(s.byte);
            if (blk == blocks - 1)
              for (int k = (blk & 3) + 1; k < 4; ++k) *++sp = 0;           // the row's last scale word
          }
        }
      }
    }
    fence_proxy_async_smem();                                             // before the next sample's copies overwrite the rows
    __syncthreads();
  }
}

// chunks per sample: all SMs busy, at least one step of rows per CTA
int chunks_of(int B, int T, int C) {
  const Lanes l = lanes_of(C);
  int P = sm_count() / B;
  const int most = (T + l.R - 1) / l.R;
  if (most <= kAloneSteps) return 1;
  if (P > most) P = most;
  if (P > 32 * kPartsPerLane) P = 32 * kPartsPerLane;
  return P < 1 ? 1 : P;
}

template <typename T, int MODE, int COLS>
int launch_norm(NormArgs a, cudaStream_t st) {
  const int longest = (a.T + a.P - 1) / a.P;
  const int fixed = smem_of(a.C, a.groups, 0).total + 256;
  const int most = fixed < kSmemMax ? (kSmemMax - fixed) / (a.C * 2 + 4) : 0;     // rows of the ring
  a.l = lanes_of(a.C);
  // segments of whole steps of R rows where that leaves all rows in the ring, then of a quarter of the rows, then of a quarter
  // of the ring
  const int R = a.l.R, quarter = (longest + kSlots - 1) / kSlots, steps = (quarter + R - 1) / R * R;
  auto ring = [&](int rows) { return (longest + rows - 1) / rows * rows; };
  int seg = ring(steps) <= most ? steps : (ring(quarter) <= most ? quarter : most / kSlots);
  if (ring(seg) > most && seg > R) seg = seg / R * R;
  if (seg < 1) return PQ_ERR_UNSUPPORTED;                                  // thousands of groups of thousands of channels
  if (MODE != kOut16 && static_cast<int64_t>(seg) * kSlots < longest) return PQ_ERR_UNSUPPORTED;      // rows beyond the chip's shared memory
  a.seg_rows = seg;
  const int slots = (longest + seg - 1) / seg < kSlots ? (longest + seg - 1) / seg : kSlots;
  a.chunk = a.T / a.P; a.longer = a.T % a.P;
  a.lay = smem_of(a.C, a.groups, slots * seg);
  if (a.lay.total > kSmemMax) return PQ_ERR_UNSUPPORTED;
  a.cpg = a.C / a.groups; a.inv_cpg = 1.0f / static_cast<float>(a.cpg);
  a.inv_cols = 1.0f / static_cast<float>(a.l.cols); a.inv_R = 1.0f / static_cast<float>(a.l.R);
  a.nch = a.C >> 4; a.R2 = a.nch > 0 ? kThreads / a.nch : 0; a.inv_nch = a.nch > 0 ? 1.0f / static_cast<float>(a.nch) : 0.0f;
  auto kern = pq_group_norm_kernel<T, MODE, COLS>;
  static bool attr_set[64] = {false};     // per device; benign race: the attribute value never changes
  int dev = 0;
  PQ_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    PQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int sms = sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.P), static_cast<unsigned>(a.B < sms ? a.B : sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(a.lay.total);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.P > 1 ? 1 : 0;                                         // nobody waits for another CTA otherwise
  PQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a));
  return PQ_OK;
}

template <int MODE>
int group_norm_any(const void* x, int dtype, int64_t B, int64_t T, int64_t C, int64_t ld_row, int64_t ld_batch, int groups,
                   const void* gamma, const void* beta, int affine_fp32, float eps, int act, void* out, int64_t ldo_row,
                   int64_t ldo_batch, uint8_t* codes, uint8_t* scales, float* row_scale, void* workspace, int64_t ws_bytes,
                   void* status, void* stream) {
  if (B < 0 || T < 0 || C <= 0 || groups <= 0 || B > 65535 || T > 0x7fffffffLL || C > kMaxC || C % groups != 0) return PQ_ERR_SHAPE;
  if (!(eps >= 0.0f) || ld_row < C || ld_batch < 0 || (out != nullptr && (ldo_row < C || ldo_batch < 0))) return PQ_ERR_SHAPE;
  if (dtype != PQ_DTYPE_BF16 && dtype != PQ_DTYPE_FP16) return PQ_ERR_DTYPE;
  if (act != PQ_ACT_NONE && act != PQ_ACT_SILU) return PQ_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return PQ_OK;
  if (x == nullptr || workspace == nullptr || (MODE == kOut16 && out == nullptr)) return PQ_ERR_NULL;
  if (MODE != kOut16 && (codes == nullptr || (MODE != kMx && row_scale == nullptr) || (MODE >= kMx && scales == nullptr))) return PQ_ERR_NULL;
  if (C % (MODE == kOut16 ? 8 : (MODE == kInt8 ? 16 : 32)) != 0 || ld_row % 8 != 0 || ld_batch % 8 != 0) return PQ_ERR_ALIGN;
  if (out != nullptr && (ldo_row % 8 != 0 || ldo_batch % 8 != 0 || !aligned_to(out, 16))) return PQ_ERR_ALIGN;
  if (!aligned_to(x, 16) || !aligned_to(workspace, 8) || !aligned_to(gamma, 16) || !aligned_to(beta, 16) || !aligned_to(codes, 16) || !aligned_to(scales, 16) || !aligned_to(row_scale, 4))
    return PQ_ERR_ALIGN;
  if (ws_bytes < pq_group_norm_workspace_bytes(B, T, C, groups)) return PQ_ERR_WORKSPACE;
  NormArgs a{};
  a.x = x; a.ld_row = ld_row; a.ld_batch = ld_batch; a.gamma = gamma; a.beta = beta; a.affine_f32 = affine_fp32 != 0;
  a.out = out; a.out_row = ldo_row; a.out_batch = ldo_batch; a.codes = codes; a.scales = scales; a.row_scale = row_scale;
  a.part = static_cast<float2*>(workspace); a.status = static_cast<int32_t*>(status);
  a.B = static_cast<int>(B); a.T = static_cast<int>(T); a.C = static_cast<int>(C); a.groups = groups;
  a.P = chunks_of(a.B, a.T, a.C); a.silu = act == PQ_ACT_SILU; a.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (lanes_of(a.C).ncol > kThreads)
    return dtype == PQ_DTYPE_BF16 ? launch_norm<__nv_bfloat16, MODE, 2>(a, st) : launch_norm<__half, MODE, 2>(a, st);
  return dtype == PQ_DTYPE_BF16 ? launch_norm<__nv_bfloat16, MODE, 1>(a, st) : launch_norm<__half, MODE, 1>(a, st);
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
                             void* out, int64_t ldo_row, int64_t ldo_batch, void* workspace, int64_t ws_bytes, void* status,
                             void* stream) {
  return group_norm_any<kOut16>(x, dtype, B, T, C, ld_row, ld_batch, groups, gamma, beta, affine_fp32, eps, act, out, ldo_row,
                                ldo_batch, nullptr, nullptr, nullptr, workspace, ws_bytes, status, stream);
}

extern "C" int pq_group_norm_quant_rows(const void* x, int dtype, int64_t B, int64_t T, int64_t C, int64_t ld_row,
                                        int64_t ld_batch, int groups, const void* gamma, const void* beta, int affine_fp32,
                                        float eps, int act, void* x_norm, int64_t ldn_row, int64_t ldn_batch, int8_t* q, float* s,
                                        void* workspace, int64_t ws_bytes, void* status, void* stream) {
  return group_norm_any<kInt8>(x, dtype, B, T, C, ld_row, ld_batch, groups, gamma, beta, affine_fp32, eps, act, x_norm, ldn_row,
                               ldn_batch, reinterpret_cast<uint8_t*>(q), nullptr, s, workspace, ws_bytes, status, stream);
}

extern "C" int pq_group_norm_quant_fp4(const void* x, int dtype, int64_t B, int64_t T, int64_t C, int64_t ld_row,
                                       int64_t ld_batch, int groups, const void* gamma, const void* beta, int affine_fp32,
                                       float eps, int act, int fmt, uint8_t* codes, uint8_t* scales, float* row_scale,
                                       void* workspace, int64_t ws_bytes, void* status, void* stream) {
  if (fmt == PQ_FP4_MX)
    return group_norm_any<kMx>(x, dtype, B, T, C, ld_row, ld_batch, groups, gamma, beta, affine_fp32, eps, act, nullptr, 0, 0, codes,
                               scales, row_scale, workspace, ws_bytes, status, stream);
  if (fmt == PQ_FP4_NV)
    return group_norm_any<kNv>(x, dtype, B, T, C, ld_row, ld_batch, groups, gamma, beta, affine_fp32, eps, act, nullptr, 0, 0, codes,
                               scales, row_scale, workspace, ws_bytes, status, stream);
  return PQ_ERR_UNSUPPORTED;
}
