// The norms before and after a transformer block with its gate and residual
// scale, forward and backward, for sm_100a. For each row of `cols` elements:
//
//   q = 1 / sqrt(mean(x^2) + eps)          p = x q post_weight  (p = x without post_weight)
//   h = residual_scale residual + gate p   (gate = 1 without one)
//   t = 1 / sqrt(mean(h^2) + eps)          n = h t weight
//
// x is the block's output, h the new residual stream, n the next block's input.
// All of it is fp32; h and n are each rounded once (n from the unrounded h).
// Backward, from dn and dh (either may be missing = zero), with xh = x q, hh = h t:
//
//   a  = dn weight                   m1 = mean(a hh)
//   D  = dh + t (a - hh m1)          d residual = residual_scale D
//   c  = gate D post_weight          m2 = mean(c xh)
//   dx = q (c - xh m2)               (dx = gate D without post_weight)
//   d weight = sum_rows dn hh, d post_weight = sum_rows gate D xh, d gate = sum D p
//
// HBM-bound: forward reads x and residual and writes n and h, backward reads x,
// residual, dn and dh and writes dx and d residual; q and t are kept from the
// forward pass (8 bytes a row), h is recomputed rather than read back rounded.
//
// Each row needs two sums over the row, the second of values that the first
// scales, so a kernel that loads a row, reduces, and loads the next leaves the
// memory idle unless other rows are in flight. Forward has one row for each
// group of kTpr threads and enough CTAs on an SM. Backward holds the parameters'
// sums in registers, so few CTAs fit; they are persistent and stream their rows
// through a ring in shared memory filled by bulk copies, so the next rows arrive
// while this one is reduced. Rows that are not whole 16-byte units, or not
// aligned to them, take the same passes element by element (simple kernels);
// rows longer than 16384 16-bit or 8192 fp32 elements (backward: 8192) take
// looping kernels that read their row again.
//
// The parameters' gradients are sums over rows. Each backward CTA walks a
// fixed range of rows ("slot") and keeps its sums in registers; slots are
// written as fp32 partials and a second launch adds them in a fixed order, so
// results do not vary from run to run (no atomics).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "cf_common.cuh"
#include "ptx.cuh"
#include "row_ring.cuh"

namespace cfb {
namespace {

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements moved as one access of up to 16 bytes at a time.
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

// How a row is spread over threads: chunk i of thread t starts at column
// (i * kTpr + t) * kVec, so a warp's accesses are contiguous.
template <int kElems, int kPerAccess>
struct Spread {
  static constexpr int kPer = kElems;        // elements per thread
  static constexpr int kVec = kPerAccess;    // elements per access
  static constexpr int kChunks = kPer / kVec;
};
// Rows of 16-byte units: 16 elements a thread, 8 of fp32.
template <typename T>
using Wide = Spread<sizeof(T) == 4 ? 8 : 16, 16 / static_cast<int>(sizeof(T))>;
// The simple kernels hold four values and three sums of each element.
using Simple = Spread<8, 1>;

template <typename T, int kVec>
__device__ __forceinline__ void load_vec(const T *p, float *f) {
  const Pack<T, kVec> v = *reinterpret_cast<const Pack<T, kVec> *>(p);
#pragma unroll
  for (int e = 0; e < kVec; ++e) f[e] = to_float<T>(v.v[e]);
}

template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T *p, const float *f) {
  Pack<T, kVec> v;
#pragma unroll
  for (int e = 0; e < kVec; ++e) v.v[e] = from_float<T>(f[e]);
  *reinterpret_cast<Pack<T, kVec> *>(p) = v;
}

// The kernels for rows of 16-byte units work on pairs of floats with packed arithmetic: at 16 bits
// an element these kernels are otherwise bound by instruction issue (84
// instructions an element backward, 36 forward, before this; see the kernels).
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) { return {ptx::pack_f32x2(lo, hi)}; }
__device__ __forceinline__ Pair both(float v) { return {ptx::splat_f32x2(v)}; }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) { return {ptx::mul_f32x2(a.v, b.v)}; }
__device__ __forceinline__ Pair operator+(Pair a, Pair b) { return {ptx::add_f32x2(a.v, b.v)}; }
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  return {ptx::fma_f32x2(a.v, b.v, c.v)};
}
__device__ __forceinline__ float sum(Pair a) {
  const float2 f = ptx::unpack_f32x2(a.v);
  return f.x + f.y;
}

// 16 bytes of T as pairs.
template <typename T>
__device__ __forceinline__ Pair widen(uint32_t two);
template <>
__device__ __forceinline__ Pair widen<__nv_bfloat16>(uint32_t two) {
  return pair(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
template <>
__device__ __forceinline__ Pair widen<__half>(uint32_t two) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&two));
  return pair(f.x, f.y);
}

template <typename T, int kPairs>
__device__ __forceinline__ void widen(const uint4 &v, Pair (&f)[kPairs]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = pair(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = pair(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    f[0] = widen<T>(v.x);
    f[1] = widen<T>(v.y);
    f[2] = widen<T>(v.z);
    f[3] = widen<T>(v.w);
  }
}

// kVec elements (16 bytes of 16-bit elements, or any whole number of float4s).
template <typename T, int kVec>
__device__ __forceinline__ void load_pairs(const T *p, Pair (&f)[kVec / 2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kVec / 4; ++i) {
      const float4 v = reinterpret_cast<const float4 *>(p)[i];
      f[2 * i] = pair(v.x, v.y);
      f[2 * i + 1] = pair(v.z, v.w);
    }
  } else {
    static_assert(kVec == 8, "one 16-byte access");
    widen<T>(*reinterpret_cast<const uint4 *>(p), f);
  }
}

template <typename T, int kVec>
__device__ __forceinline__ void store_pairs(T *p, const Pair (&f)[kVec / 2]) {
  float2 v[kVec / 2];
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) v[i] = ptx::unpack_f32x2(f[i].v);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kVec / 4; ++i) {
      reinterpret_cast<float4 *>(p)[i] =
          make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
    }
  } else {
    static_assert(kVec == 8, "one 16-byte access");
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = std::is_same_v<T, __half> ? ptx::pack_f16x2(v[i].x, v[i].y)
                                       : ptx::pack_bf16x2(v[i].x, v[i].y);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Sum over the kTpr threads of a row. Groups of one warp need no barrier;
// wider groups are the whole CTA and alternate between two buffers, so one
// barrier per sum suffices (the next write of a buffer comes after the barrier
// of the sum in between, which every reader of this one has passed).
template <int kTpr>
__device__ __forceinline__ float row_sum(float v, float (*buf)[32], int &parity) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (kTpr > kWarp) {
    constexpr int kWarps = kTpr / kWarp;
    const int lane = threadIdx.x & (kWarp - 1);
    if (lane == 0) buf[parity][threadIdx.x / kWarp] = v;
    __syncthreads();
    v = lane < kWarps ? buf[parity][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    parity ^= 1;
  }
  return v;
}

struct NormArgs {
  const void *x, *residual, *weight, *post, *gate;
  void *n, *h;
  float *stats;  // [rows][2]: q and t, or null
  int64_t rows, cols;
  int64_t gate_rows;  // rows that share a row of the gate
  float scale, eps;
  // backward
  const void *dn, *dh;
  void *dx, *dres, *dgate;
  float *part;  // partial sums: [3][slots][cols] (weight, post, gate)
  float *means; // [rows][2]: m1 and m2 (long rows)
  int64_t slots, group_chunks, rows_per_slot;
  bool whole_groups;  // a slot holds whole gate groups and writes their gradients itself
  // staged kernels
  int stages;
  unsigned *err;
};

constexpr int kThreadsSmall = 128;  // CTA of the warp-per-row form: four rows

template <int kTpr>
constexpr int cta_threads() { return kTpr == kWarp ? kThreadsSmall : kTpr; }

// ---------------------------------------------------------------- forward

// One row for each group of threads, in registers through both passes. What
// hides a row's two sums is other CTAs' rows, so registers are what bounds it:
// inputs stay packed, and 1536 threads fit on an SM. [16384, 4096] bf16 with a
// gate: 87 us, 6.2 TB/s (1024 threads 97 us; unpacked scalar arithmetic 108 us;
// persistent CTAs with the backward kernel's ring 122 us).
template <typename T, typename TW, int kTpr>
__global__ void __launch_bounds__(cta_threads<kTpr>(), 1536 / cta_threads<kTpr>())
    gated_norm_kernel(const NormArgs a) {
  using S = Wide<T>;
  constexpr int kPairs = S::kVec / 2;
  __shared__ float buf[2][32];
  int parity = 0;
  constexpr int kRows = cta_threads<kTpr>() / kTpr;
  const int t = threadIdx.x % kTpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTpr;
  if (row >= a.rows) return;  // whole warps, and only where a row is one warp
  const int cols = static_cast<int>(a.cols);
  const float inv_cols = 1.0f / static_cast<float>(cols);
  const T *x = static_cast<const T *>(a.x) + row * a.cols;
  const T *r = static_cast<const T *>(a.residual) + row * a.cols;
  const TW *weight = static_cast<const TW *>(a.weight);
  const TW *post = static_cast<const TW *>(a.post);
  const TW *gate = a.gate ? static_cast<const TW *>(a.gate) + row / a.gate_rows * a.cols : nullptr;
  // The inputs stay packed until they are used: more CTAs fit on an SM.
  uint4 xr[S::kChunks], rr[S::kChunks];
  Pair h[S::kChunks][kPairs], ss = both(0.0f);
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
    const int c = (i * kTpr + t) * S::kVec;
    if (c < cols) {
      xr[i] = *reinterpret_cast<const uint4 *>(x + c);
      rr[i] = *reinterpret_cast<const uint4 *>(r + c);
    }
  }
  float q = 1.0f;
  if (post != nullptr) {
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      if ((i * kTpr + t) * S::kVec < cols) {
        Pair p[kPairs];
        widen<T>(xr[i], p);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) ss = fma(p[e], p[e], ss);
      }
    }
    q = rsqrtf(row_sum<kTpr>(sum(ss), buf, parity) * inv_cols + a.eps);
    ss = both(0.0f);
  }
  const Pair q2 = both(q), scale2 = both(a.scale);
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
    const int c = (i * kTpr + t) * S::kVec;
    if (c < cols) {
      Pair p[kPairs], w[kPairs];
      widen<T>(xr[i], p);
      widen<T>(rr[i], h[i]);
      if (post != nullptr) {
        load_pairs<TW, S::kVec>(post + c, w);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) p[e] = p[e] * q2 * w[e];
      }
      if (gate != nullptr) {
        load_pairs<TW, S::kVec>(gate + c, w);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) p[e] = p[e] * w[e];
      }
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        h[i][e] = fma(scale2, h[i][e], p[e]);
        ss = fma(h[i][e], h[i][e], ss);
      }
      store_pairs<T, S::kVec>(static_cast<T *>(a.h) + row * a.cols + c, h[i]);
    }
  }
  const float rt = rsqrtf(row_sum<kTpr>(sum(ss), buf, parity) * inv_cols + a.eps);
  const Pair rt2 = both(rt);
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
    const int c = (i * kTpr + t) * S::kVec;
    if (c < cols) {
      Pair w[kPairs];
      load_pairs<TW, S::kVec>(weight + c, w);
#pragma unroll
      for (int e = 0; e < kPairs; ++e) w[e] = h[i][e] * rt2 * w[e];
      store_pairs<T, S::kVec>(static_cast<T *>(a.n) + row * a.cols + c, w);
    }
  }
  if (a.stats != nullptr && t == 0) {
    a.stats[2 * row] = q;
    a.stats[2 * row + 1] = rt;
  }
}

// The same passes with the row in registers, element by element, one row for
// each group of threads.
template <typename T, typename TW, int kTpr>
__global__ void __launch_bounds__(cta_threads<kTpr>())
    gated_norm_simple_kernel(const NormArgs a) {
  using S = Simple;
  __shared__ float buf[2][32];
  int parity = 0;
  constexpr int kRows = cta_threads<kTpr>() / kTpr;
  const int t = threadIdx.x % kTpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTpr;
  if (row >= a.rows) return;  // whole warps, and only where a row is one warp
  const int cols = static_cast<int>(a.cols);
  const T *x = static_cast<const T *>(a.x) + row * a.cols;
  const T *r = static_cast<const T *>(a.residual) + row * a.cols;
  const TW *weight = static_cast<const TW *>(a.weight);
  const TW *post = static_cast<const TW *>(a.post);
  const TW *gate = a.gate ? static_cast<const TW *>(a.gate) + row / a.gate_rows * a.cols : nullptr;
  float xv[S::kPer], rv[S::kPer];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
    const int c = (i * kTpr + t) * S::kVec;
    if (c < cols) {
      load_vec<T, S::kVec>(x + c, xv + i * S::kVec);
      load_vec<T, S::kVec>(r + c, rv + i * S::kVec);
    } else {
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) xv[i * S::kVec + e] = rv[i * S::kVec + e] = 0.0f;
    }
  }
  const float inv_cols = 1.0f / static_cast<float>(cols);
  float q = 1.0f;
  if (post != nullptr) {
#pragma unroll
    for (int e = 0; e < S::kPer; ++e) sum = fmaf(xv[e], xv[e], sum);
    q = rsqrtf(row_sum<kTpr>(sum, buf, parity) * inv_cols + a.eps);
  }
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
    const int c = (i * kTpr + t) * S::kVec;
    if (c < cols) {
      float *h = rv + i * S::kVec;
      float p[S::kVec], w[S::kVec];
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) p[e] = xv[i * S::kVec + e] * q;
      if (post != nullptr) {
        load_vec<TW, S::kVec>(post + c, w);
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) p[e] *= w[e];
      }
      if (gate != nullptr) {
        load_vec<TW, S::kVec>(gate + c, w);
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) p[e] *= w[e];
      }
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) {
        h[e] = fmaf(a.scale, h[e], p[e]);
        sum = fmaf(h[e], h[e], sum);
      }
      store_vec<T, S::kVec>(static_cast<T *>(a.h) + row * a.cols + c, h);
    }
  }
  const float rt = rsqrtf(row_sum<kTpr>(sum, buf, parity) * inv_cols + a.eps);
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
    const int c = (i * kTpr + t) * S::kVec;
    if (c < cols) {
      float w[S::kVec], n[S::kVec];
      load_vec<TW, S::kVec>(weight + c, w);
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) n[e] = rv[i * S::kVec + e] * rt * w[e];
      store_vec<T, S::kVec>(static_cast<T *>(a.n) + row * a.cols + c, n);
    }
  }
  if (a.stats != nullptr && t == 0) {
    a.stats[2 * row] = q;
    a.stats[2 * row + 1] = rt;
  }
}

// Element c of a row's residual sum, and of p, in fp32 (long rows: recomputed
// in each pass).
template <typename T, typename TW>
__device__ __forceinline__ float sum_at(const NormArgs &a, const T *x, const T *r, const TW *gate,
                                        int64_t c, float q, float &xh, float &p) {
  xh = to_float<T>(x[c]) * q;
  p = a.post ? xh * to_float<TW>(static_cast<const TW *>(a.post)[c]) : xh;
  const float g = gate ? to_float<TW>(gate[c]) * p : p;
  return fmaf(a.scale, to_float<T>(r[c]), g);
}

constexpr int kLongThreads = 1024;

template <typename T, typename TW>
__global__ void __launch_bounds__(kLongThreads) gated_norm_long_kernel(const NormArgs a) {
  __shared__ float buf[2][32];
  int parity = 0;
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + row * a.cols;
  const T *r = static_cast<const T *>(a.residual) + row * a.cols;
  const TW *weight = static_cast<const TW *>(a.weight);
  const TW *gate = a.gate ? static_cast<const TW *>(a.gate) + row / a.gate_rows * a.cols : nullptr;
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  float q = 1.0f, sum = 0.0f, xh, p;
  if (a.post != nullptr) {
    for (int64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
      const float v = to_float<T>(x[c]);
      sum = fmaf(v, v, sum);
    }
    q = rsqrtf(row_sum<kLongThreads>(sum, buf, parity) * inv_cols + a.eps);
  }
  sum = 0.0f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float h = sum_at<T, TW>(a, x, r, gate, c, q, xh, p);
    static_cast<T *>(a.h)[row * a.cols + c] = from_float<T>(h);
    sum = fmaf(h, h, sum);
  }
  const float rt = rsqrtf(row_sum<kLongThreads>(sum, buf, parity) * inv_cols + a.eps);
  for (int64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float h = sum_at<T, TW>(a, x, r, gate, c, q, xh, p);
    static_cast<T *>(a.n)[row * a.cols + c] = from_float<T>(h * rt * to_float<TW>(weight[c]));
  }
  if (a.stats != nullptr && threadIdx.x == 0) {
    a.stats[2 * row] = q;
    a.stats[2 * row + 1] = rt;
  }
}

// ---------------------------------------------------------------- backward

// Rows [begin, end) of a slot. Either slots hold whole gate groups, or a group
// is cut into group_chunks slots that stay inside it.
__device__ __forceinline__ void slot_rows(const NormArgs &a, int64_t slot, int64_t group_rows,
                                          int64_t &begin, int64_t &end) {
  if (a.whole_groups) {
    begin = slot * a.rows_per_slot;
    end = min(a.rows, begin + a.rows_per_slot);
  } else {
    const int64_t group = slot / a.group_chunks;
    const int64_t first = group * group_rows;
    begin = min(first + (slot - group * a.group_chunks) * a.rows_per_slot, first + group_rows);
    end = min(begin + a.rows_per_slot, first + group_rows);
  }
}

// CTAs of the backward kernel on an SM: 512 threads at up to 128 registers (one
// CTA of 1024 threads has 64).
template <int kTpr>
constexpr int backward_ctas() {
  return cta_threads<kTpr>() > 512 ? 1 : 512 / cta_threads<kTpr>();
}

// ---------------------------------------------------------------- row ring

constexpr int kMaxStages = 4;

// All threads of a row's group.
template <int kTpr>
__device__ __forceinline__ void group_sync() {
  if constexpr (kTpr > kWarp) {
    __syncthreads();
  } else {
    __syncwarp();
  }
}

// weight and post_weight (ones without it) as fp32 in shared memory, loaded once
// by a persistent CTA. A thread reads kVec consecutive values as float4s; they
// are stored so that each of its float4s is next to its neighbours' (kVec 8: the
// first halves of all groups of eight, then the second halves), which keeps the
// accesses free of bank conflicts.
template <int kVec>
__device__ __forceinline__ int staged_at(int c, int cols) {
  return kVec == 8 ? (c & 4 ? cols / 2 : 0) + (c >> 3) * 4 + (c & 3) : c;
}

template <typename TW, int kVec>
__device__ __forceinline__ void stage_weights(float *post_s, float *weight_s, const void *post,
                                              const void *weight, int cols) {
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    const int at = staged_at<kVec>(c, cols);
    weight_s[at] = to_float<TW>(static_cast<const TW *>(weight)[c]);
    post_s[at] = post ? to_float<TW>(static_cast<const TW *>(post)[c]) : 1.0f;
  }
}

template <int kVec>
__device__ __forceinline__ void load_staged(const float *w, int c, int cols,
                                            Pair (&f)[kVec / 2]) {
#pragma unroll
  for (int i = 0; i < kVec / 4; ++i) {
    const float4 v = *reinterpret_cast<const float4 *>(w + staged_at<kVec>(c + 4 * i, cols));
    f[2 * i] = pair(v.x, v.y);
    f[2 * i + 1] = pair(v.z, v.w);
  }
}

// kShared: a row of the gate serves gate_rows > 1 rows, so its gradient is a
// sum; otherwise there is none, or one for each row. kFull: the row fills the
// group's registers exactly, so no chunk is conditional; the branches around them
// keep the compiler from interleaving the chunks. [8192, 4096] bf16 with a gate:
// 91 us (105 with the branches, 157 without the ring), 4.4 TB/s, and 8 us to add
// the partial sums; bound by latency at the 512 threads that an SM has registers
// for (half of the issue slots are taken, and two thirds of the memory's rate).
template <typename T, typename TW, int kTpr, bool kShared, bool kFull>
__global__ void __launch_bounds__(cta_threads<kTpr>(), backward_ctas<kTpr>())
    gated_norm_backward_kernel(const NormArgs a) {
  using S = Wide<T>;
  constexpr int kPairs = S::kVec / 2;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  constexpr int kSlots = cta_threads<kTpr>() / kTpr;
  __shared__ float buf[2][32];
  __shared__ __align__(8) uint64_t full[kSlots][kMaxStages];
  int parity = 0;
  const int in_cta = threadIdx.x / kTpr;
  const int t = threadIdx.x % kTpr;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * kSlots + in_cta;
  const int cols = kFull ? kTpr * S::kPer : static_cast<int>(a.cols);
  const float inv_cols = 1.0f / static_cast<float>(cols);
  float *post_s = reinterpret_cast<float *>(smem_raw);
  float *weight_s = post_s + cols;
  int64_t begin = 0, end = 0;
  if (slot < a.slots) slot_rows(a, slot, kShared ? a.gate_rows : a.rows, begin, end);

  RowRing<4> ring;
  ring.src[0] = static_cast<const uint8_t *>(a.x);
  ring.src[1] = static_cast<const uint8_t *>(a.residual);
  ring.src[2] = static_cast<const uint8_t *>(a.dn);
  ring.src[3] = static_cast<const uint8_t *>(a.dh);
  ring.row_bytes = static_cast<uint32_t>(cols * sizeof(T));
  ring.stages = a.stages;
  ring.smem = smem_raw + 2 * cols * sizeof(float) +
              static_cast<size_t>(in_cta) * a.stages * 4 * ring.row_bytes;
  ring.full = full[in_cta];
  ring.err = a.err;
  if (t == 0) {
    ring.init();
    for (int s = 0; s < a.stages && begin + s < end; ++s) ring.issue(s, begin + s);
  }
  stage_weights<TW, S::kVec>(post_s, weight_s, a.post, a.weight, cols);
  __syncthreads();
  if (slot >= a.slots) return;  // whole warps, and only where a row is one warp

  Pair sum_w[S::kChunks][kPairs], sum_p[S::kChunks][kPairs], sum_g[S::kChunks][kPairs];
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
#pragma unroll
    for (int e = 0; e < kPairs; ++e) sum_w[i][e] = sum_p[i][e] = sum_g[i][e] = both(0.0f);
  }
  // Two loads: a caller's stats need no more than a float's alignment.
  auto stats_of = [&](int64_t row) { return make_float2(a.stats[2 * row], a.stats[2 * row + 1]); };
  float2 stats = begin < end ? stats_of(begin) : float2{};
  const Pair scale2 = both(a.scale);

  for (int64_t row = begin; row < end; ++row) {
    const int64_t base = row * a.cols;
    const TW *gate = a.gate == nullptr ? nullptr
                                       : static_cast<const TW *>(a.gate) +
                                             (kShared ? row / a.gate_rows : row) * a.cols;
    const Pair q2 = both(stats.x), rt2 = both(stats.y);
    if (row + 1 < end) stats = stats_of(row + 1);
    ring.wait();
    const T *x = ring.template row<T>(0);
    const T *r = ring.template row<T>(1);
    const T *dn = ring.template row<T>(2);
    const T *dh = ring.template row<T>(3);

    // hh and a stay in registers for the second pass; d takes a's place there.
    Pair hh[S::kChunks][kPairs], av[S::kChunks][kPairs];
    Pair neg_m1 = both(0.0f);
    if (a.dn != nullptr) {
      Pair s1 = both(0.0f);
#pragma unroll
      for (int i = 0; i < S::kChunks; ++i) {
        const int c = (i * kTpr + t) * S::kVec;
        if (kFull || c < cols) {
          Pair p[kPairs], w[kPairs];
          load_pairs<T, S::kVec>(x + c, p);
          load_pairs<T, S::kVec>(r + c, hh[i]);
          load_staged<S::kVec>(post_s, c, cols, w);
#pragma unroll
          for (int e = 0; e < kPairs; ++e) p[e] = p[e] * q2 * w[e];
          if (gate != nullptr) {
            load_pairs<TW, S::kVec>(gate + c, w);
#pragma unroll
            for (int e = 0; e < kPairs; ++e) p[e] = p[e] * w[e];
          }
          load_staged<S::kVec>(weight_s, c, cols, w);
          load_pairs<T, S::kVec>(dn + c, av[i]);
#pragma unroll
          for (int e = 0; e < kPairs; ++e) {
            hh[i][e] = fma(scale2, hh[i][e], p[e]) * rt2;
            sum_w[i][e] = fma(av[i][e], hh[i][e], sum_w[i][e]);
            av[i][e] = av[i][e] * w[e];
            s1 = fma(av[i][e], hh[i][e], s1);
          }
        }
      }
      neg_m1 = both(-row_sum<kTpr>(sum(s1), buf, parity) * inv_cols);
    }

    Pair s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int c = (i * kTpr + t) * S::kVec;
      if (kFull || c < cols) {
        Pair xh[kPairs], w[kPairs], out[kPairs], *d = av[i];
        if (a.dh != nullptr) {
          load_pairs<T, S::kVec>(dh + c, out);
        } else {
#pragma unroll
          for (int e = 0; e < kPairs; ++e) out[e] = both(0.0f);
        }
        load_pairs<T, S::kVec>(x + c, xh);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          xh[e] = xh[e] * q2;
          d[e] = a.dn != nullptr ? fma(rt2, fma(hh[i][e], neg_m1, d[e]), out[e]) : out[e];
          out[e] = d[e] * scale2;
        }
        store_pairs<T, S::kVec>(static_cast<T *>(a.dres) + base + c, out);
        Pair pw[kPairs];
        load_staged<S::kVec>(post_s, c, cols, pw);
        if (gate != nullptr) {
          load_pairs<TW, S::kVec>(gate + c, w);
#pragma unroll
          for (int e = 0; e < kPairs; ++e) {
            out[e] = d[e] * (xh[e] * pw[e]);
            if constexpr (kShared) sum_g[i][e] = sum_g[i][e] + out[e];
            d[e] = d[e] * w[e];
          }
          if constexpr (!kShared) {
            store_pairs<TW, S::kVec>(static_cast<TW *>(a.dgate) + base + c, out);
          }
        }
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          sum_p[i][e] = fma(d[e], xh[e], sum_p[i][e]);
          d[e] = d[e] * pw[e];
          s2 = fma(d[e], xh[e], s2);
        }
      }
    }
    // Without post_weight there is no first norm: dx = d.
    Pair neg_m2 = both(0.0f);
    if (a.post != nullptr) neg_m2 = both(-row_sum<kTpr>(sum(s2), buf, parity) * inv_cols);
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int c = (i * kTpr + t) * S::kVec;
      if (kFull || c < cols) {
        Pair xh[kPairs];
        load_pairs<T, S::kVec>(x + c, xh);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) xh[e] = fma(xh[e] * q2, neg_m2, av[i][e]) * q2;
        store_pairs<T, S::kVec>(static_cast<T *>(a.dx) + base + c, xh);
      }
    }
    // The row has been read: its stage takes the row `stages` ahead.
    group_sync<kTpr>();
    if (t == 0 && row + a.stages < end) ring.issue(ring.stage, row + a.stages);
    ring.advance();
    if constexpr (kShared) {
      if (a.whole_groups && (row + 1) % a.gate_rows == 0) {
#pragma unroll
        for (int i = 0; i < S::kChunks; ++i) {
          const int c = (i * kTpr + t) * S::kVec;
          if (kFull || c < cols) {
            store_pairs<TW, S::kVec>(
                static_cast<TW *>(a.dgate) + row / a.gate_rows * a.cols + c, sum_g[i]);
          }
#pragma unroll
          for (int e = 0; e < kPairs; ++e) sum_g[i][e] = both(0.0f);
        }
      }
    }
  }
  if (t == 0) ring.drain();
  const int64_t plane = a.slots * a.cols;
  float *part = a.part + slot * a.cols;
#pragma unroll
  for (int i = 0; i < S::kChunks; ++i) {
    const int c = (i * kTpr + t) * S::kVec;
    if (kFull || c < cols) {
      store_pairs<float, S::kVec>(part + c, sum_w[i]);
      if (a.post) store_pairs<float, S::kVec>(part + plane + c, sum_p[i]);
      if (kShared && !a.whole_groups) store_pairs<float, S::kVec>(part + 2 * plane + c, sum_g[i]);
    }
  }
}

// The same with the row in registers, element by element.
template <typename T, typename TW, int kTpr, bool kShared>
__global__ void __launch_bounds__(cta_threads<kTpr>())
    gated_norm_backward_simple_kernel(const NormArgs a) {
  using S = Simple;
  __shared__ float buf[2][32];
  int parity = 0;
  constexpr int kSlots = cta_threads<kTpr>() / kTpr;
  const int t = threadIdx.x % kTpr;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * kSlots + threadIdx.x / kTpr;
  if (slot >= a.slots) return;  // whole warps, and only where a row is one warp
  const int cols = static_cast<int>(a.cols);
  const float inv_cols = 1.0f / static_cast<float>(cols);
  const TW *weight = static_cast<const TW *>(a.weight);
  const TW *post = static_cast<const TW *>(a.post);
  const int64_t group_rows = kShared ? a.gate_rows : a.rows;
  int64_t begin, end;
  slot_rows(a, slot, group_rows, begin, end);

  float sum_w[S::kPer], sum_p[S::kPer], sum_g[S::kPer];
#pragma unroll
  for (int e = 0; e < S::kPer; ++e) sum_w[e] = sum_p[e] = sum_g[e] = 0.0f;

  for (int64_t row = begin; row < end; ++row) {
    const int64_t base = row * a.cols;
    const TW *gate = a.gate == nullptr ? nullptr
                                       : static_cast<const TW *>(a.gate) +
                                             (kShared ? row / a.gate_rows : row) * a.cols;
    const float q = a.stats[2 * row], rt = a.stats[2 * row + 1];
    float xh[S::kPer], hh[S::kPer], av[S::kPer], dv[S::kPer];
    float s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int c = (i * kTpr + t) * S::kVec;
      const int o = i * S::kVec;
#pragma unroll
      for (int e = 0; e < S::kVec; ++e) xh[o + e] = hh[o + e] = av[o + e] = dv[o + e] = 0.0f;
      if (c < cols) {
        load_vec<T, S::kVec>(static_cast<const T *>(a.x) + base + c, xh + o);
        load_vec<T, S::kVec>(static_cast<const T *>(a.residual) + base + c, hh + o);
        if (a.dn) load_vec<T, S::kVec>(static_cast<const T *>(a.dn) + base + c, av + o);
        if (a.dh) load_vec<T, S::kVec>(static_cast<const T *>(a.dh) + base + c, dv + o);
      }
    }
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int c = (i * kTpr + t) * S::kVec;
      if (c < cols) {
        float w[S::kVec], p[S::kVec];
        const int o = i * S::kVec;
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) p[e] = xh[o + e] = xh[o + e] * q;
        if (post != nullptr) {
          load_vec<TW, S::kVec>(post + c, w);
#pragma unroll
          for (int e = 0; e < S::kVec; ++e) p[e] *= w[e];
        }
        if (gate != nullptr) {
          load_vec<TW, S::kVec>(gate + c, w);
#pragma unroll
          for (int e = 0; e < S::kVec; ++e) p[e] *= w[e];
        }
        load_vec<TW, S::kVec>(weight + c, w);
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) {
          hh[o + e] = fmaf(a.scale, hh[o + e], p[e]) * rt;
          sum_w[o + e] = fmaf(av[o + e], hh[o + e], sum_w[o + e]);
          av[o + e] *= w[e];
          s1 = fmaf(av[o + e], hh[o + e], s1);
        }
      }
    }
    const float m1 = row_sum<kTpr>(s1, buf, parity) * inv_cols;
    float s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int c = (i * kTpr + t) * S::kVec;
      if (c < cols) {
        const int o = i * S::kVec;
        float w[S::kVec], d[S::kVec], out[S::kVec];
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) {
          d[e] = fmaf(rt, fmaf(-hh[o + e], m1, av[o + e]), dv[o + e]);
          out[e] = a.scale * d[e];
        }
        store_vec<T, S::kVec>(static_cast<T *>(a.dres) + base + c, out);
        float pw[S::kVec];
        if (post != nullptr) load_vec<TW, S::kVec>(post + c, pw);
        if (gate != nullptr) {
          load_vec<TW, S::kVec>(gate + c, w);
#pragma unroll
          for (int e = 0; e < S::kVec; ++e) {
            out[e] = d[e] * xh[o + e];
            if (post != nullptr) out[e] *= pw[e];
            if constexpr (kShared) sum_g[o + e] += out[e];
            d[e] *= w[e];
          }
          if constexpr (!kShared) {
            store_vec<TW, S::kVec>(static_cast<TW *>(a.dgate) + base + c, out);
          }
        }
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) {
          if (post != nullptr) {
            sum_p[o + e] = fmaf(d[e], xh[o + e], sum_p[o + e]);
            d[e] *= pw[e];
            s2 = fmaf(d[e], xh[o + e], s2);
          }
          dv[o + e] = d[e];
        }
      }
    }
    float m2 = 0.0f;
    if (post != nullptr) m2 = row_sum<kTpr>(s2, buf, parity) * inv_cols;
    const bool group_done = kShared && a.whole_groups && (row + 1) % a.gate_rows == 0;
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int c = (i * kTpr + t) * S::kVec;
      if (c < cols) {
        const int o = i * S::kVec;
        float out[S::kVec];
#pragma unroll
        for (int e = 0; e < S::kVec; ++e) {
          out[e] = post != nullptr ? q * fmaf(-xh[o + e], m2, dv[o + e]) : dv[o + e];
        }
        store_vec<T, S::kVec>(static_cast<T *>(a.dx) + base + c, out);
        if constexpr (kShared) {
          if (group_done) {
            store_vec<TW, S::kVec>(
                static_cast<TW *>(a.dgate) + row / a.gate_rows * a.cols + c, sum_g + o);
#pragma unroll
            for (int e = 0; e < S::kVec; ++e) sum_g[o + e] = 0.0f;
          }
        }
      }
    }
  }
  // Partial sums; a slot without rows leaves zeros.
  const int64_t plane = a.slots * a.cols;
  float *part = a.part + slot * a.cols;
#pragma unroll
  for (int i = 0; i < S::kPer; ++i) {
    const int c = i * kTpr + t;
    if (c < cols) {
      part[c] = sum_w[i];
      if (post != nullptr) part[plane + c] = sum_p[i];
      if (kShared && !a.whole_groups) part[2 * plane + c] = sum_g[i];
    }
  }
}

// Long rows: m1 and m2 of each row with dx and d residual, then the columns'
// sums in a kernel of their own.
template <typename T, typename TW>
__global__ void __launch_bounds__(kLongThreads) gated_norm_backward_long_kernel(const NormArgs a) {
  __shared__ float buf[2][32];
  int parity = 0;
  const int64_t row = blockIdx.x;
  const int64_t base = row * a.cols;
  const T *x = static_cast<const T *>(a.x) + base;
  const T *r = static_cast<const T *>(a.residual) + base;
  const T *dn = a.dn ? static_cast<const T *>(a.dn) + base : nullptr;
  const T *dh = a.dh ? static_cast<const T *>(a.dh) + base : nullptr;
  const TW *weight = static_cast<const TW *>(a.weight);
  const TW *post = static_cast<const TW *>(a.post);
  const TW *gate = a.gate ? static_cast<const TW *>(a.gate) + row / a.gate_rows * a.cols : nullptr;
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const float q = a.stats[2 * row], rt = a.stats[2 * row + 1];
  float s = 0.0f, m1 = 0.0f, m2 = 0.0f, xh, p;
  if (dn) {
    for (int64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
      const float hh = sum_at<T, TW>(a, x, r, gate, c, q, xh, p) * rt;
      s = fmaf(to_float<T>(dn[c]) * to_float<TW>(weight[c]), hh, s);
    }
    m1 = row_sum<kLongThreads>(s, buf, parity) * inv_cols;
  }
  s = 0.0f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
      const float hh = sum_at<T, TW>(a, x, r, gate, c, q, xh, p) * rt;
      const float av = dn ? to_float<T>(dn[c]) * to_float<TW>(weight[c]) : 0.0f;
      float d = fmaf(rt, fmaf(-hh, m1, av), dh ? to_float<T>(dh[c]) : 0.0f);
      if (pass == 0) {
        static_cast<T *>(a.dres)[base + c] = from_float<T>(a.scale * d);
        if (gate && a.gate_rows == 1) static_cast<TW *>(a.dgate)[base + c] = from_float<TW>(d * p);
      }
      if (gate) d *= to_float<TW>(gate[c]);
      if (post) d *= to_float<TW>(post[c]);
      if (pass == 0) {
        s = fmaf(d, xh, s);
      } else {
        static_cast<T *>(a.dx)[base + c] =
            from_float<T>(post ? q * fmaf(-xh, m2, d) : d);
      }
    }
    if (pass == 0 && post) m2 = row_sum<kLongThreads>(s, buf, parity) * inv_cols;
  }
  if (threadIdx.x == 0) {
    a.means[2 * row] = m1;
    a.means[2 * row + 1] = m2;
  }
}

constexpr int kColumnThreads = 256;

template <typename T, typename TW>
__global__ void __launch_bounds__(kColumnThreads)
    gated_norm_backward_columns_kernel(const NormArgs a) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kColumnThreads + threadIdx.x;
  if (c >= a.cols) return;
  const bool shared_gate = a.gate != nullptr && a.gate_rows > 1;
  const int64_t slot = blockIdx.y;
  int64_t begin, end;
  slot_rows(a, slot, shared_gate ? a.gate_rows : a.rows, begin, end);
  float sum_w = 0.0f, sum_p = 0.0f, sum_g = 0.0f;
  const float w = to_float<TW>(static_cast<const TW *>(a.weight)[c]);
  for (int64_t row = begin; row < end; ++row) {
    const int64_t base = row * a.cols;
    const TW *gate =
        a.gate ? static_cast<const TW *>(a.gate) + row / a.gate_rows * a.cols : nullptr;
    const float q = a.stats[2 * row], rt = a.stats[2 * row + 1];
    float xh, p;
    const float hh = sum_at<T, TW>(a, static_cast<const T *>(a.x) + base,
                                   static_cast<const T *>(a.residual) + base, gate, c, q, xh, p) *
                     rt;
    const float dn = a.dn ? to_float<T>(static_cast<const T *>(a.dn)[base + c]) : 0.0f;
    const float dh = a.dh ? to_float<T>(static_cast<const T *>(a.dh)[base + c]) : 0.0f;
    const float d = fmaf(rt, fmaf(-hh, a.means[2 * row], dn * w), dh);
    sum_w = fmaf(dn, hh, sum_w);
    sum_g = fmaf(d, p, sum_g);
    sum_p = fmaf(gate ? d * to_float<TW>(gate[c]) : d, xh, sum_p);
    if (shared_gate && a.whole_groups && (row + 1) % a.gate_rows == 0) {
      static_cast<TW *>(a.dgate)[row / a.gate_rows * a.cols + c] = from_float<TW>(sum_g);
      sum_g = 0.0f;
    }
  }
  const int64_t plane = a.slots * a.cols;
  float *part = a.part + slot * a.cols + c;
  part[0] = sum_w;
  if (a.post) part[plane] = sum_p;
  if (shared_gate && !a.whole_groups) part[2 * plane] = sum_g;
}

// Adds the slots' partial sums. blockIdx.y: 0 weight, 1 post_weight, 2 + g the
// gate's group g. A thread adds every kFinishRows-th slot, in order.
constexpr int kFinishCols = 32, kFinishRows = 32;

template <typename TW>
__global__ void __launch_bounds__(kFinishCols *kFinishRows)
    gated_norm_finish_kernel(const float *part, int64_t slots, int64_t cols, int64_t group_chunks,
                             TW *dweight, TW *dpost, TW *dgate) {
  __shared__ float sums[kFinishRows][kFinishCols + 1];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kFinishCols + threadIdx.x;
  const int64_t which = blockIdx.y;
  TW *out = which == 0 ? dweight : which == 1 ? dpost : dgate + (which - 2) * cols;
  if (which == 1 && dpost == nullptr) return;
  const int64_t first = which < 2 ? 0 : (which - 2) * group_chunks;
  const int64_t count = which < 2 ? slots : group_chunks;
  const float *src = part + (min(which, int64_t{2}) * slots + first) * cols + c;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t k = threadIdx.y; k < count; k += kFinishRows) s += src[k * cols];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < kFinishRows; ++k) total += sums[k][threadIdx.x];
    out[c] = from_float<TW>(total);
  }
}

// ---------------------------------------------------------------- host

// Threads for a row of `cols` elements at `per` elements a thread; 0: long row.
int threads_per_row(int64_t cols, int per) {
  for (int tpr : {32, 64, 128, 256, 512, 1024}) {
    if (cols <= static_cast<int64_t>(tpr) * per) return tpr;
  }
  return 0;
}

// The longest row of the staged and simple backward kernels.
constexpr int64_t kBackwardMaxCols = 8192;

// The backward pass's slots: as many rows at a time as an SM holds (512 threads of
// them), since more only add partial sums.
void plan_slots(NormArgs &a, int dtype, bool shared_gate) {
  const int tpr =
      a.cols > kBackwardMaxCols ? 0 : threads_per_row(a.cols, dtype == CF_DTYPE_F32 ? 8 : 16);
  const int64_t per_sm = tpr == 0 ? 2 : std::max(1, 512 / tpr);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(a.rows, per_sm * sm_count()));
  const int64_t group_rows = shared_gate ? a.gate_rows : a.rows;
  const int64_t groups = a.rows / group_rows;
  if (shared_gate && groups >= want) {
    a.whole_groups = true;
    a.group_chunks = 1;
    const int64_t per_slot = (groups + want - 1) / want;
    a.rows_per_slot = per_slot * group_rows;
    a.slots = (groups + per_slot - 1) / per_slot;
  } else {
    a.whole_groups = false;
    a.group_chunks = std::min(group_rows, std::max<int64_t>(1, want / groups));
    a.rows_per_slot = (group_rows + a.group_chunks - 1) / a.group_chunks;
    a.group_chunks = (group_rows + a.rows_per_slot - 1) / a.rows_per_slot;
    a.slots = groups * a.group_chunks;
  }
}

size_t part_bytes(const NormArgs &a, bool post, bool shared_gate) {
  const size_t planes = shared_gate && !a.whole_groups ? 3 : post ? 2 : 1;
  const size_t bytes = planes * static_cast<size_t>(a.slots) * static_cast<size_t>(a.cols) * 4;
  return (bytes + 255) & ~static_cast<size_t>(255);
}

// Stages of a ring whose CTA holds `groups` of them beside its two fp32 weight
// rows, with `ctas` such CTAs on an SM: as many as fit, up to kMaxStages.
constexpr int64_t kRingSmem = int64_t{216} << 10;  // an SM has 227 KB for CTAs
int ring_stages(int arrays, int64_t cols, int64_t elem, int groups, int ctas) {
  const int64_t left = kRingSmem / ctas - 2 * cols * 4;
  return static_cast<int>(
      std::min<int64_t>(kMaxStages, std::max<int64_t>(0, left) / (arrays * cols * elem * groups)));
}

template <auto Kernel>
int launch_staged(NormArgs a, int arrays, int64_t elem, int groups, unsigned grid, int threads,
                  int ctas, cudaStream_t s) {
  while (ctas > 1 && ring_stages(arrays, a.cols, elem, groups, ctas) < 2) ctas /= 2;
  a.stages = ring_stages(arrays, a.cols, elem, groups, ctas);
  if (a.stages < 1) return CF_ERR_UNSUPPORTED;  // not for any length the kernels are built for
  a.err = device_error_word();
  if (a.err == nullptr) return record_cuda_error(cudaGetLastError());
  const size_t smem =
      2 * a.cols * 4 + static_cast<size_t>(a.stages) * arrays * a.cols * elem * groups;
  if (int st = allow_dynamic_smem<Kernel>(kRingSmem)) return st;
  Kernel<<<grid, threads, smem, s>>>(a);
  return check_launch();
}

template <typename T, typename TW, int kTpr>
int launch_forward(const NormArgs &a, bool wide, cudaStream_t s) {
  constexpr int kRows = cta_threads<kTpr>() / kTpr;
  const unsigned grid = static_cast<unsigned>((a.rows + kRows - 1) / kRows);
  if (wide) {
    gated_norm_kernel<T, TW, kTpr><<<grid, cta_threads<kTpr>(), 0, s>>>(a);
  } else {
    gated_norm_simple_kernel<T, TW, kTpr><<<grid, cta_threads<kTpr>(), 0, s>>>(a);
  }
  return check_launch();
}

template <typename T, typename TW>
int forward(const NormArgs &a, bool wide, cudaStream_t s) {
  switch (threads_per_row(a.cols, wide ? Wide<T>::kPer : Simple::kPer)) {
    case 32: return launch_forward<T, TW, 32>(a, wide, s);
    case 64: return launch_forward<T, TW, 64>(a, wide, s);
    case 128: return launch_forward<T, TW, 128>(a, wide, s);
    case 256: return launch_forward<T, TW, 256>(a, wide, s);
    case 512: return launch_forward<T, TW, 512>(a, wide, s);
    case 1024: return launch_forward<T, TW, 1024>(a, wide, s);
    default:
      gated_norm_long_kernel<T, TW>
          <<<static_cast<unsigned>(a.rows), kLongThreads, 0, s>>>(a);
      return check_launch();
  }
}

template <bool kShared, bool kFull>
struct BackwardForm {
  static constexpr bool shared = kShared, full = kFull;
};

template <typename T, typename TW, int kTpr>
int launch_backward(const NormArgs &a, bool wide, cudaStream_t s) {
  constexpr int kThreads = cta_threads<kTpr>();
  constexpr int kSlots = kThreads / kTpr;
  const unsigned grid = static_cast<unsigned>((a.slots + kSlots - 1) / kSlots);
  const bool shared = a.gate != nullptr && a.gate_rows > 1;
  if (!wide) {
    if (shared) {
      gated_norm_backward_simple_kernel<T, TW, kTpr, true><<<grid, kThreads, 0, s>>>(a);
    } else {
      gated_norm_backward_simple_kernel<T, TW, kTpr, false><<<grid, kThreads, 0, s>>>(a);
    }
    return check_launch();
  }
  // The staged kernel's widest group covers kBackwardMaxCols.
  constexpr int kWideTpr =
      std::min<int>(kTpr, static_cast<int>(kBackwardMaxCols / Wide<T>::kPer));
  constexpr int ctas = backward_ctas<kWideTpr>();
  auto run = [&](auto tag) {
    return launch_staged<gated_norm_backward_kernel<T, TW, kWideTpr, decltype(tag)::shared,
                                                    decltype(tag)::full>>(
        a, 4, sizeof(T), kSlots, grid, kThreads, ctas, s);
  };
  const bool full = a.cols == kWideTpr * Wide<T>::kPer;
  if (shared) return full ? run(BackwardForm<true, true>{}) : run(BackwardForm<true, false>{});
  return full ? run(BackwardForm<false, true>{}) : run(BackwardForm<false, false>{});
}

template <typename T, typename TW>
int backward(const NormArgs &a, bool wide, void *dweight, void *dpost, cudaStream_t s) {
  int st = CF_OK;
  switch (a.cols > kBackwardMaxCols
              ? 0
              : threads_per_row(a.cols, wide ? Wide<T>::kPer : Simple::kPer)) {
#define CFB_CASE(tpr)                              \
  case tpr:                                        \
    st = launch_backward<T, TW, tpr>(a, wide, s);  \
    break
    CFB_CASE(32);
    CFB_CASE(64);
    CFB_CASE(128);
    CFB_CASE(256);
    CFB_CASE(512);
    CFB_CASE(1024);
#undef CFB_CASE
    default: {
      gated_norm_backward_long_kernel<T, TW>
          <<<static_cast<unsigned>(a.rows), kLongThreads, 0, s>>>(a);
      if ((st = check_launch()) != CF_OK) return st;
      const dim3 grid(static_cast<unsigned>((a.cols + kColumnThreads - 1) / kColumnThreads),
                      static_cast<unsigned>(a.slots));
      gated_norm_backward_columns_kernel<T, TW><<<grid, kColumnThreads, 0, s>>>(a);
      st = check_launch();
    }
  }
  if (st != CF_OK) return st;
  const bool gate_parts = a.gate != nullptr && a.gate_rows > 1 && !a.whole_groups;
  const dim3 grid(static_cast<unsigned>((a.cols + kFinishCols - 1) / kFinishCols),
                  static_cast<unsigned>(2 + (gate_parts ? a.slots / a.group_chunks : 0)));
  gated_norm_finish_kernel<TW><<<grid, dim3(kFinishCols, kFinishRows), 0, s>>>(
      a.part, a.slots, a.cols, a.group_chunks, static_cast<TW *>(dweight),
      static_cast<TW *>(dpost), static_cast<TW *>(a.dgate));
  return check_launch();
}

template <bool kForward>
int dispatch_norm(const NormArgs &a, int dtype, int weight_dtype, bool wide, void *dweight,
                  void *dpost, cudaStream_t s) {
  const bool wf = weight_dtype == CF_DTYPE_F32;
#define CFB_RUN(T, TW)                                       \
  do {                                                       \
    if constexpr (kForward) {                                \
      return forward<T, TW>(a, wide, s);                     \
    } else {                                                 \
      return backward<T, TW>(a, wide, dweight, dpost, s);    \
    }                                                        \
  } while (0)
  switch (dtype) {
    case CF_DTYPE_F32: CFB_RUN(float, float);
    case CF_DTYPE_BF16:
      if (wf) CFB_RUN(__nv_bfloat16, float);
      CFB_RUN(__nv_bfloat16, __nv_bfloat16);
    default:
      if (wf) CFB_RUN(__half, float);
      CFB_RUN(__half, __half);
  }
#undef CFB_RUN
}

// Checks shared by both directions.
int check_norm_args(int64_t rows, int64_t cols, int64_t gate_groups, bool gate, int dtype,
                    int weight_dtype) {
  if (rows < 0 || cols < 0 || (gate && gate_groups < (rows > 0 ? 1 : 0))) {
    return CF_ERR_INVALID_ARGUMENT;
  }
  if (dtype != CF_DTYPE_F32 && dtype != CF_DTYPE_BF16 && dtype != CF_DTYPE_F16) {
    return CF_ERR_UNSUPPORTED;
  }
  if (weight_dtype != dtype && weight_dtype != CF_DTYPE_F32) return CF_ERR_UNSUPPORTED;
  if (rows == 0 || cols == 0) return CF_OK;
  if (gate && rows % gate_groups != 0) return CF_ERR_INVALID_ARGUMENT;
  // Grid dimensions: rows in x, gate groups and slots in y.
  if (rows > 0x7fffffffll || cols > (int64_t{1} << 40) / rows) return CF_ERR_INVALID_ARGUMENT;
  return CF_OK;
}

bool wide_rows(int64_t cols, int dtype, std::initializer_list<const void *> pointers) {
  if (cols % (dtype == CF_DTYPE_F32 ? 4 : 8) != 0) return false;
  for (const void *p : pointers) {
    if (!aligned_to(p, 16)) return false;  // a null pointer is aligned
  }
  return true;
}

}  // namespace
}  // namespace cfb

extern "C" {

int cf_gated_residual_rmsnorm(const void *x, const void *residual, const void *weight,
                              const void *post_weight, const void *gate, int64_t gate_groups,
                              int weight_dtype, void *normalised, void *residual_out, float *stats,
                              int64_t rows, int64_t cols, float residual_scale, float eps,
                              int dtype, cf_stream_t stream) {
  if (int st = cfb::check_norm_args(rows, cols, gate_groups, gate != nullptr, dtype,
                                    weight_dtype)) {
    return st;
  }
  if (rows == 0 || cols == 0) return CF_OK;
  if (!x || !residual || !weight || !normalised || !residual_out) return CF_ERR_INVALID_ARGUMENT;
  cfb::NormArgs a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.post = post_weight;
  a.gate = gate;
  a.gate_rows = gate ? rows / gate_groups : rows;
  a.n = normalised;
  a.h = residual_out;
  a.stats = stats;
  a.rows = rows;
  a.cols = cols;
  a.scale = residual_scale;
  a.eps = eps;
  const bool wide = cfb::wide_rows(
      cols, dtype, {x, residual, weight, post_weight, gate, normalised, residual_out});
  return cfb::dispatch_norm<true>(a, dtype, weight_dtype, wide, nullptr, nullptr,
                             reinterpret_cast<cudaStream_t>(stream));
}

size_t cf_gated_residual_rmsnorm_backward_workspace_bytes(int64_t rows, int64_t cols,
                                                          int has_post_weight,
                                                          int64_t gate_groups, int dtype) {
  if (rows <= 0 || cols <= 0 || (gate_groups > 0 && rows % gate_groups != 0)) return 0;
  cfb::NormArgs a{};
  a.rows = rows;
  a.cols = cols;
  const bool shared = gate_groups > 0 && gate_groups < rows;
  a.gate_rows = gate_groups > 0 ? rows / gate_groups : rows;
  cfb::plan_slots(a, dtype, shared);
  size_t bytes = cfb::part_bytes(a, has_post_weight != 0, shared);
  if (cols > cfb::kBackwardMaxCols) {
    bytes += static_cast<size_t>(rows) * 2 * sizeof(float);
  }
  return bytes;
}

int cf_gated_residual_rmsnorm_backward(
    const void *d_normalised, const void *d_residual_out, const void *x, const void *residual,
    const void *weight, const void *post_weight, const void *gate, int64_t gate_groups,
    int weight_dtype, const float *stats, void *dx, void *d_residual, void *d_weight,
    void *d_post_weight, void *d_gate, int64_t rows, int64_t cols, float residual_scale, int dtype,
    void *workspace, size_t workspace_bytes, cf_stream_t stream) {
  if (int st = cfb::check_norm_args(rows, cols, gate_groups, gate != nullptr, dtype,
                                    weight_dtype)) {
    return st;
  }
  if (rows == 0 || cols == 0) return CF_OK;
  if (!x || !residual || !weight || !stats || !dx || !d_residual || !d_weight ||
      (d_post_weight == nullptr) != (post_weight == nullptr) ||
      (d_gate == nullptr) != (gate == nullptr)) {
    return CF_ERR_INVALID_ARGUMENT;
  }
  cfb::NormArgs a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.post = post_weight;
  a.gate = gate;
  a.gate_rows = gate ? rows / gate_groups : rows;
  a.stats = const_cast<float *>(stats);
  a.rows = rows;
  a.cols = cols;
  a.scale = residual_scale;
  a.dn = d_normalised;
  a.dh = d_residual_out;
  a.dx = dx;
  a.dres = d_residual;
  a.dgate = d_gate;
  const bool shared = gate != nullptr && a.gate_rows > 1;
  cfb::plan_slots(a, dtype, shared);
  const size_t need = cf_gated_residual_rmsnorm_backward_workspace_bytes(
      rows, cols, post_weight != nullptr, gate ? gate_groups : 0, dtype);
  if (workspace == nullptr || workspace_bytes < need) return CF_ERR_WORKSPACE;
  if (!cfb::aligned_to(workspace, 16)) return CF_ERR_MISALIGNED;
  a.part = static_cast<float *>(workspace);
  a.means = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                      cfb::part_bytes(a, post_weight != nullptr, shared));
  const bool wide = cfb::wide_rows(cols, dtype,
                                   {x, residual, weight, post_weight, gate, dx, d_residual,
                                    d_normalised, d_residual_out, d_gate});
  return cfb::dispatch_norm<false>(a, dtype, weight_dtype, wide, d_weight, d_post_weight,
                              reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
