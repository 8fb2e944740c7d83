// 8-bit floating-point (e4m3) quantisation with a scale for each block of 128,
// and the matrix product of operands held that way, for sm_100a.
//
//   scale = fl32(absmax * fl32(1 / 448)), 1 when not > 0 (zero, NaN, underflow)
//   code  = e4m3(fl32(x / scale)), nearest even, saturating at +-448, NaN kept
// over blocks of 1 x 128 (activations) or 128 x 128 (weights); the last block of
// a row may be shorter. The product of a [m, k] in 1 x 128 blocks and b [n, k]
// in 128 x 128 blocks is
//   y[m, n] = sum_kb a_scale[m, kb] b_scale[n / 128, kb] (sum_{k in kb} a[m, k] b[n, k])
// The inner sums are exact products accumulated in fp32 by the tensor core; the
// outer sum is fp32 in registers: scales are arbitrary fp32 numbers, so they
// cannot ride on the MMA's own power-of-two block scales.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "cf_common.cuh"
#include "gemm_common.cuh"
#include "ptx.cuh"
#include "stage_ring.cuh"
#include "stream.cuh"

namespace cfb {
namespace {

constexpr int kBlock = CF_FP8_BLOCK_SIZE;
constexpr float kInvE4m3Max = 1.0f / 448.0f;

// ---------------------------------------------------------------- quantisation

// Scale of a block from the bit pattern of its absmax (a NaN's is the largest).
__device__ __forceinline__ float fp8_scale(unsigned absmax_bits) {
  const float s = __fmul_rn(__uint_as_float(absmax_bits), kInvE4m3Max);
  return s > 0.0f ? s : 1.0f;
}

// Whether x / s may be formed as in fp8_quotient for every element of a block: s
// far enough from the ends of the range that the residual x - q s is exact for
// every quotient that does not round to zero, and no infinity or NaN.
__device__ __forceinline__ bool fp8_fast(unsigned absmax_bits, float s) {
  return absmax_bits < 0x7f800000u && s >= 0x1p-60f && s <= 0x1p100f;
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight elements to eight codes. fl32(x / s) without a division, two at a time: r
// = fl32(1 / s), q0 = fl(x r), the exact residual and Markstein's correction step
// (as quant_math.cuh). The residual is rounded downwards, which being exact it does
// not notice, except that a zero is -0 then: added to q0 = -0, the quotient of x = -0,
// a +0 would lose the sign.
__device__ __forceinline__ uint2 fp8_codes(const float (&f)[8], float s, float r, bool fast) {
  float q[8];
  if (fast) {
    const uint64_t r2 = ptx::splat_f32x2(r), neg_s2 = ptx::splat_f32x2(-s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t x2 = ptx::pack_f32x2(f[2 * i], f[2 * i + 1]);
      const uint64_t q0 = ptx::mul_f32x2(x2, r2);
      const float2 v =
          ptx::unpack_f32x2(ptx::fma_f32x2(ptx::fma_down_f32x2(q0, neg_s2, x2), r2, q0));
      q[2 * i] = v.x;
      q[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(f[i], s);
  }
  return make_uint2(e4m3x2(q[0], q[1]) | e4m3x2(q[2], q[3]) << 16,
                    e4m3x2(q[4], q[5]) | e4m3x2(q[6], q[7]) << 16);
}

template <typename T>
__device__ __forceinline__ float as_float(T v) {
  if constexpr (std::is_same_v<T, float>) {
    return v;
  } else if constexpr (std::is_same_v<T, __half>) {
    return __half2float(v);
  } else {
    return __bfloat162float(v);
  }
}

// Eight consecutive elements as they are stored, and their absmax's bit pattern
// as an fp32 number (magnitudes of one type order as their bits do, a NaN's
// highest). 16-bit elements stay packed: two a compare.
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }

  // `left` of the eight are inside the row, the rest are zeros. kWide: p is on a
  // 16-byte boundary and left is not between 0 and 8.
  template <bool kWide>
  __device__ __forceinline__ void load(const T *p, int left) {
    zero();
    if constexpr (kWide) {
      if (left <= 0) return;
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
      T *e = reinterpret_cast<T *>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i < left) e[i] = p[i];
      }
    }
  }

  // Largest magnitude, packed: the bits of one fp32, or of two 16-bit halves.
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      m = larger(m, w[i] & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu));
    }
    return m;
  }

  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b);
  }

  static __device__ __forceinline__ unsigned bits(uint32_t top) {
    if constexpr (sizeof(T) == 4) {
      return top;
    } else {
      const uint16_t h = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
      return __float_as_uint(as_float<T>(*reinterpret_cast<const T *>(&h)));
    }
  }

  __device__ __forceinline__ void widen(float (&f)[8]) const {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = as_float<T>(e[i]);
    }
  }

  __device__ __forceinline__ uint2 codes(float s, float r, bool fast) const {
    float f[8];
    widen(f);
    return fp8_codes(f, s, r, fast);
  }
};

template <bool kWide>
__device__ __forceinline__ void store8(uint8_t *p, int left, uint2 codes) {
  if constexpr (kWide) {
    if (left > 0) *reinterpret_cast<uint2 *>(p) = codes;
  } else {
    const uint8_t *b = reinterpret_cast<const uint8_t *>(&codes);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < left) p[i] = b[i];
    }
  }
}

constexpr int kQuantThreads = 256;
// Longest row: a CTA's offsets from its first row are 32-bit.
constexpr int64_t kQuantMaxCols = int64_t{1} << 30;
// Blocks in flight for each half-warp (at [8192, 4096] fp32, two: 29 us, four: 33;
// at [8192, 11008] bf16, two: 63, four: 58).
template <typename T>
constexpr int kQuantUnroll = sizeof(T) == 4 ? 2 : 4;

// 1 x 128 blocks: 16 lanes a block, eight elements a lane; kUnroll blocks a
// half-warp, loaded before any is reduced. [8192, 11008] bf16: 58 us, 4.6 TB/s, bound
// by latency at the 1024 threads that an SM has registers for, a warp's loads and its
// arithmetic taking turns (two thirds of the issue slots are taken, and of the memory's
// rate; fp32, half the instructions a byte: 5.8). Everything beyond
// a CTA's first block is 32-bit offsets: at 16 bits an element 64-bit addresses were a
// third of the instructions, and their registers half of the CTAs that fit on an SM.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kQuantThreads, 4)
    fp8_quantize_rows_kernel(const T *x, uint8_t *codes, float *scales, int64_t blocks, int cols,
                             int row_blocks, int64_t scale_row, int64_t scale_kb) {
  constexpr int kUnroll = kQuantUnroll<T>;
  constexpr int kStride = kQuantThreads / 16;
  ptx::grid_dep_launch_dependents();  // a product may fetch its weights meanwhile
  const int lane16 = threadIdx.x & 15;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kStride * kUnroll);
  const int64_t row0 = blocks <= 0xffffffffll
                           ? static_cast<uint32_t>(first) / static_cast<uint32_t>(row_blocks)
                           : first / row_blocks;
  const int here = static_cast<int>(min(blocks - first, int64_t{kStride * kUnroll}));
  x += row0 * cols;
  codes += row0 * cols;
  scales += row0 * scale_row;
  // (row, kb): this half-warp's block, rows counted from the CTA's first.
  int row = 0, kb = static_cast<int>(first - row0 * row_blocks) + threadIdx.x / 16;
  Eight<T> v[kUnroll];
  int rows[kUnroll], kbs[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    while (kb >= row_blocks) {
      kb -= row_blocks;
      ++row;
    }
    rows[u] = row;
    kbs[u] = kb;
    const int c = kb * kBlock + lane16 * 8;
    const bool in = static_cast<int>(u * kStride + threadIdx.x / 16) < here;
    v[u].template load<kWide>(x + (row * cols + c), in ? cols - c : 0);
    kb += kStride;
  }
  // Each lane takes the scale of one of its half-warp's blocks, not of all.
  uint32_t mine = 0;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    uint32_t top = v[u].top();
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      top = Eight<T>::larger(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if ((lane16 & (kUnroll - 1)) == u) mine = top;
  }
  const unsigned m = Eight<T>::bits(mine);
  const float my_scale = fp8_scale(m);
  const float my_inverse = fp8_fast(m, my_scale) ? __frcp_rn(my_scale) : 0.0f;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const float s = __shfl_sync(0xffffffffu, my_scale, u, 16);
    const float r = __shfl_sync(0xffffffffu, my_inverse, u, 16);
    const int c = kbs[u] * kBlock + lane16 * 8;
    const bool in = static_cast<int>(u * kStride + threadIdx.x / 16) < here;
    store8<kWide>(codes + (rows[u] * cols + c), in ? cols - c : 0,
                  v[u].codes(s, r, r != 0.0f));
    if (lane16 == 0 && in) scales[rows[u] * scale_row + kbs[u] * scale_kb] = s;
  }
}

// 128 x 128 blocks: one CTA each, eight rows of eight elements a thread. [11008,
// 4096] bf16: 24 us, 5.7 TB/s.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 4 ? 2 : 4)
    fp8_quantize_blocks_kernel(const T *x, uint8_t *codes, float *scales, int64_t rows, int cols) {
  constexpr int kRowsAtOnce = kQuantThreads / 16;
  constexpr int kSteps = kBlock / kRowsAtOnce;
  __shared__ uint32_t warp_top[kQuantThreads / kWarp];
  const int c = blockIdx.x * kBlock + (threadIdx.x & 15) * 8;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kBlock + threadIdx.x / 16;
  const int left = cols - c;
  // Rows of this thread that exist.
  const int steps = static_cast<int>(
      min(int64_t{kSteps}, max(int64_t{0}, (rows - r0 + kRowsAtOnce - 1) / kRowsAtOnce)));
  const int64_t stride = static_cast<int64_t>(kRowsAtOnce) * cols;
  Eight<T> v[kSteps];
  uint32_t top = 0;
  const T *from = x + r0 * cols + c;
#pragma unroll
  for (int i = 0; i < kSteps; ++i, from += stride) {
    v[i].template load<kWide>(from, i < steps ? left : 0);
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) top = Eight<T>::larger(top, v[i].top());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = Eight<T>::larger(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if ((threadIdx.x & (kWarp - 1)) == 0) warp_top[threadIdx.x / kWarp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / kWarp; ++w) top = Eight<T>::larger(top, warp_top[w]);
  const unsigned m = Eight<T>::bits(top);
  const float s = fp8_scale(m);
  const bool fast = fp8_fast(m, s);
  const float inv = fast ? __frcp_rn(s) : 0.0f;
  uint8_t *to = codes + r0 * cols + c;
#pragma unroll
  for (int i = 0; i < kSteps; ++i, to += stride) {
    store8<kWide>(to, i < steps ? left : 0, v[i].codes(s, inv, fast));
  }
  if (threadIdx.x == 0) scales[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

template <typename T>
int quantize_fp8(const void *x, uint8_t *codes, float *scales, int64_t rows, int64_t cols,
                 int block_rows, int64_t scale_pitch, cudaStream_t s) {
  const T *in = static_cast<const T *>(x);
  const bool wide = cols % 8 == 0 && aligned_to(x, 16) && aligned_to(codes, 8);
  const int64_t row_blocks = (cols + kBlock - 1) / kBlock;
  if (block_rows == 1) {
    const int64_t blocks = rows * row_blocks;
    const int64_t per_cta = kQuantThreads / 16 * kQuantUnroll<T>;
    const int64_t grid = (blocks + per_cta - 1) / per_cta;
    if (grid > 0x7fffffffll) return CF_ERR_INVALID_ARGUMENT;
    const int64_t scale_row = scale_pitch > 0 ? 1 : row_blocks;
    const int64_t scale_kb = scale_pitch > 0 ? scale_pitch : 1;
    if (wide) {
      fp8_quantize_rows_kernel<T, true><<<static_cast<unsigned>(grid), kQuantThreads, 0, s>>>(
          in, codes, scales, blocks, static_cast<int>(cols), static_cast<int>(row_blocks),
          scale_row, scale_kb);
    } else {
      fp8_quantize_rows_kernel<T, false><<<static_cast<unsigned>(grid), kQuantThreads, 0, s>>>(
          in, codes, scales, blocks, static_cast<int>(cols), static_cast<int>(row_blocks),
          scale_row, scale_kb);
    }
    return check_launch();
  }
  // Bands of at most 65535 row blocks (the grid's limit in y).
  for (int64_t r = 0; r < rows; r += int64_t{65535} * kBlock) {
    const int64_t n = std::min<int64_t>(rows - r, int64_t{65535} * kBlock);
    const dim3 grid(static_cast<unsigned>(row_blocks),
                    static_cast<unsigned>((n + kBlock - 1) / kBlock));
    float *to = scales + r / kBlock * row_blocks;
    if (wide) {
      fp8_quantize_blocks_kernel<T, true>
          <<<grid, kQuantThreads, 0, s>>>(in + r * cols, codes + r * cols, to, n,
                                          static_cast<int>(cols));
    } else {
      fp8_quantize_blocks_kernel<T, false>
          <<<grid, kQuantThreads, 0, s>>>(in + r * cols, codes + r * cols, to, n,
                                          static_cast<int>(cols));
    }
    if (int st = check_launch()) return st;
  }
  return CF_OK;
}

// scale_pitch > 0: the scales of 1 x 128 blocks as [kb][scale_pitch], which is how
// the products read them, instead of [rows][kb].
int quantize_fp8_any(const void *x, int dtype, uint8_t *codes, float *scales, int64_t rows,
                     int64_t cols, int block_rows, int64_t scale_pitch, cudaStream_t s) {
  switch (dtype) {
    case CF_DTYPE_F32:
      return quantize_fp8<float>(x, codes, scales, rows, cols, block_rows, scale_pitch, s);
    case CF_DTYPE_BF16:
      return quantize_fp8<__nv_bfloat16>(x, codes, scales, rows, cols, block_rows,
                                         scale_pitch, s);
    default:
      return quantize_fp8<__half>(x, codes, scales, rows, cols, block_rows, scale_pitch, s);
  }
}

// ---------------------------------------------------------------- products

struct Fp8Params {
  const uint8_t *a;      // codes [m, k]
  const float *a_scales; // [kb][a_pitch], a row's at its index
  int64_t a_pitch;
  const uint8_t *b;      // codes [n, k]
  const float *b_scales; // [ceil(n / 128), kb]
  void *y;               // [m, n]
  int64_t m, n, k;
  int num_kb;
  int m_tiles, n_tiles, band;
  int splits;  // CTAs that share a tile's blocks of k
  int a_rows;  // rows of a in a stage: fewer than a tile's where m ends before
  bool after_quantise;  // a's codes come from the kernel launched just before
  unsigned *err;
};

// Few rows: the streaming kernel with m16n8k32 on e4m3, a block is one of the
// scales' 128 elements of k.
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T>
struct Fp8StreamOp {
  static constexpr int kMatrices = 1, kBlocks = kStreamWarps, kBlockElems = kBlock;
  static constexpr int kScaleBytes = kStreamWarps * kStreamTokens * 4;
  // Of the block of the tile's first feature and of the next: a lane holds one of the
  // next 32 steps.
  struct Weights {
    float w[2];
  };

  StreamMap w[1], less[1], tokens;
  CUtensorMap tm_scale;
  Fp8Params p;
  unsigned *err;
  StreamTiles tiles;
  int steps, whole_steps, blocks, token_rows, scale_bytes;

  __device__ __forceinline__ void load_scales(uint8_t *dst, uint64_t *bar, int step) const {
    ptx::tma_load_2d(dst, &tm_scale, bar, 0, step * kStreamWarps);
  }

  __device__ __forceinline__ void fetch(Weights &l, int feature, int step, int warp) const {
    const int64_t kb = int64_t{step + static_cast<int>(threadIdx.x % kWarp)} * kStreamWarps + warp;
    const int last_block = static_cast<int>((p.n - 1) / kBlock);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int block = min(feature / kBlock + h, last_block);
      if (kb < p.num_kb) l.w[h] = __ldg(p.b_scales + int64_t{block} * p.num_kb + kb);
    }
  }

  __device__ __forceinline__ void multiply(const StreamRows &r, const uint4 (&x)[2],
                                           const float (&s)[2], const Weights &l, int feature,
                                           int step, float (&acc)[4]) const {
    float d[2][4] = {};  // two chains of two
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mma_e4m3(d[h], r.w[0][h].x, r.w[1][h].x, r.w[0][h].y, r.w[1][h].y, x[h].x, x[h].y);
      mma_e4m3(d[h], r.w[0][h].z, r.w[1][h].z, r.w[0][h].w, r.w[1][h].w, x[h].z, x[h].w);
    }
    const float first = __shfl_sync(0xffffffffu, l.w[0], step % kWarp);
    const float second = __shfl_sync(0xffffffffu, l.w[1], step % kWarp);
    const int in_block = feature % kBlock + static_cast<int>(threadIdx.x % kWarp) / 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // the lane's features, rows g and g + 8
      const float w = in_block + i / 2 * 8 < kBlock ? first : second;
      acc[i] = fmaf(s[i & 1] * w, d[0][i] + d[1][i], acc[i]);
    }
  }

  __device__ __forceinline__ void store(int feature, int count, const float *red) const {
    if (threadIdx.x >= kStreamTokens * kStreamFeatures) return;
    const int m = threadIdx.x / kStreamFeatures, f = threadIdx.x % kStreamFeatures;
    const int64_t n = int64_t{feature} + f;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kStreamWarps; ++w) v += red[(w * kStreamTokens + m) * kStreamRedRow + f];
    if (m < p.m && f < count && n < p.n) {
      T *y = static_cast<T *>(p.y) + m * p.n + n;
      if constexpr (std::is_same_v<T, __half>) {
        *y = __float2half_rn(v);
      } else {
        *y = __float2bfloat16_rn(v);
      }
    }
  }
};

template <typename T>
int launch_fp8_stream(const Fp8Params &p, cudaStream_t s) {
  Fp8StreamOp<T> op;
  op.p = p;
  op.err = device_error_word();
  if (op.err == nullptr) return record_cuda_error(cudaGetLastError());
  op.tiles = stream_tiles(p.n);
  op.blocks = p.num_kb;
  op.steps = (p.num_kb + kStreamWarps - 1) / kStreamWarps;
  op.token_rows = static_cast<int>(p.m);
  op.whole_steps = stream_whole_steps(p.k, kStreamWarps);
  const int scale_rows = std::min(kStreamWarps, p.num_kb);
  op.scale_bytes = scale_rows * kStreamTokens * 4;
  if (int st = make_map(&op.tm_scale, p.a_scales, 4, p.m, p.num_kb, kStreamTokens, scale_rows,
                        false, p.a_pitch)) {
    return st;
  }
  auto map = [&](StreamMap &to, const uint8_t *base, int64_t n, int rows) {
    return to.make(base, 1, p.k, n, rows, kStreamWarps, op.whole_steps);
  };
  if (int st = map(op.tokens, p.a, p.m, op.token_rows)) return st;
  if (int st = map(op.w[0], p.b, p.n, op.tiles.rows)) return st;
  if (int st = map(op.less[0], p.b, p.n, std::max(1, op.tiles.rows - 1))) return st;
  return launch_stream(op, p.after_quantise, s);
}

// Many rows: tiles on tcgen05, 128 tokens a CTA and kN features. One MMA group
// of four (K = 32 each) covers a 128-block of k into one of several TMEM buffers;
// epilogue warps (a thread is a token and kThreadCols of the tile's features)
// read each finished block, multiply by a_scale b_scale and add into registers
// while the next blocks are computed.
//
// What bounds it is the way from a finished block to a free buffer (barrier,
// TMEM load, additions, barrier), since TMEM holds two blocks and registers hold
// 256 features' sums and an eighth of a block. At [16384, 8192] x [28672, 8192]
// the MMAs alone take 2.4 ms (3.2 PFLOP/s), the additions 0.6 ms on top. (192
// features, read at once and the buffer freed before any addition, were no
// faster.) So everything else is kept off these warps: the tokens' scales come by
// TMA with each stage's operands (loading them from global memory cost 0.4 ms),
// and results leave through shared memory and TMA (row by row from the threads
// that hold them, 32 rows an instruction, cost 0.25 ms). kCtas = 2: CTA pairs,
// 256 tokens, each CTA staging half of b's rows.
constexpr int kTileM = 128;
template <int kCtas, int kN>
struct TileCfg {
  // Eight epilogue warps: fewer and wider threads have fewer instructions around
  // the additions (sixteen warps of 64 columns were 4 % slower).
  static constexpr int kEpilogueWarps = 8;
  static constexpr int kThreadCols = kN / 2;
  static constexpr int kThreads = 32 * (kEpilogueWarps + 4);  // + producer, MMA, two idle
  // 168 registers a thread at launch; 128 columns' sums need more, which the other
  // warps give up (2 * 216 + 72 = 3 * 168).
  static constexpr bool kMoveRegs = kThreadCols == 128;
  static constexpr int kEpilogueRegs = 216, kOtherRegs = 72;
  static constexpr int kAtOnce = kMoveRegs ? 32 : kThreadCols;  // columns read at once
  static constexpr int kBRows = kN / kCtas;
  static constexpr int kABytes = kTileM * kBlock;
  static constexpr int kOperandBytes = kABytes + kBRows * kBlock;
  static constexpr int kScaleBytes = kTileM * 4;
  static constexpr int kOutBytes = 32 * 64;  // a warp's 32 rows x 32 columns on their way out
  static constexpr int kBuffers = 512 / kN < 4 ? 512 / kN : 4;
  static constexpr int kTmemCols = kBuffers * kN <= 256 ? 256 : 512;
  static constexpr int kStages = 6;
  // A stage's scales are read by the epilogue, after its operands' slot is free
  // again: the producer's next use of a scale slot has to come after that. It
  // refills operand slot s once the MMAs of kStages blocks ago retired, and those
  // began once the block kBuffers before them had left its TMEM buffer, scales
  // read. So this many slots need no barrier of their own.
  static constexpr int kScaleSlots = kStages + kBuffers;
  static constexpr int kOutOffset = kStages * kOperandBytes;
  static constexpr int kScaleOffset = kOutOffset + kEpilogueWarps * kOutBytes;
  static constexpr int kBarOffset = kScaleOffset + kScaleSlots * kScaleBytes;
  static constexpr size_t kSmem = 1024 + kBarOffset + 256;
  static_assert(kSmem <= 232448, "227 KB of shared memory");
};

template <int kCtas, int kN, bool kBf16, bool kSplit>
__global__ void __launch_bounds__(TileCfg<kCtas, kN>::kThreads, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap tm_a,
                    const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_scale,
                    const __grid_constant__ CUtensorMap tm_y, const Fp8Params p) {
  using C = TileCfg<kCtas, kN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::kBarOffset);
  uint64_t *empty = full + C::kStages;
  uint64_t *tmem_full = empty + C::kStages;
  uint64_t *tmem_empty = tmem_full + C::kBuffers;
  uint64_t *drain = tmem_empty + C::kBuffers;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  int *abort_flag = reinterpret_cast<int *>(tmem_slot + 1);
  const int warp = threadIdx.x / kWarp;
  const int lane = threadIdx.x % kWarp;
  static_assert(!kSplit || kCtas == 1, "a cluster is a pair or shares a tile's k");
  const uint32_t rank = kCtas == 2 ? ptx::cluster_ctarank() : 0;
  const int tiles = p.m_tiles * p.n_tiles;
  const int share = kSplit ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int first = blockIdx.x / (kSplit ? p.splits : kCtas);
  const int step = kSplit ? tiles : gridDim.x / kCtas;
  const int kb_begin = kSplit ? p.num_kb * share / p.splits : 0;
  const int kb_end = kSplit ? p.num_kb * (share + 1) / p.splits : p.num_kb;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < C::kBuffers; ++i) {
      ptx::mbar_init(&tmem_full[i], 1);
      ptx::mbar_init(&tmem_empty[i], kCtas * C::kEpilogueWarps);
    }
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == C::kEpilogueWarps && lane == 0) {
    ptx::prefetch_tensor_map(&tm_a);
    ptx::prefetch_tensor_map(&tm_b);
    ptx::prefetch_tensor_map(&tm_scale);
  }
  if (warp == C::kEpilogueWarps + 1) {
    if constexpr (kCtas == 2) {
      ptx::tmem_alloc_pair(tmem_slot, C::kTmemCols);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, C::kTmemCols);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (kCtas == 2) ptx::cluster_sync();  // both CTAs' barriers are ready
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if constexpr (C::kMoveRegs) {
    if (warp >= C::kEpilogueWarps) ptx::lower_registers<C::kOtherRegs>();
  }
  if (warp == C::kEpilogueWarps) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      ptx::grid_dep_wait();  // the tokens' codes and scales
      StageRing<C::kStages> ring;
      int slot = 0;
      for (int tile = first; tile < tiles && !aborted(abort_flag); tile += step) {
        int tm, tn;
        band_order(tile, p.m_tiles, p.n_tiles, p.band, tm, tn);
        const int a_row = (tm * kCtas + static_cast<int>(rank)) * kTileM;
        const int b_row = tn * kN + static_cast<int>(rank) * C::kBRows;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!ring.wait_free(empty)) {
            record_timeout(p.err, abort_flag);
            break;
          }
          uint64_t *const landed = &full[ring.stage];
          uint8_t *sa = smem + ring.stage * C::kOperandBytes;
          uint8_t *scale = smem + C::kScaleOffset + slot * C::kScaleBytes;
          const uint32_t bytes =
              C::kOperandBytes + C::kScaleBytes - (kTileM - p.a_rows) * kBlock;
          if constexpr (kCtas == 2) {
            // The even CTA's barrier counts both CTAs' bytes.
            const uint32_t bar = ptx::map_shared_rank(ptx::smem_addr(landed), 0);
            if (rank == 0) ptx::mbar_expect_tx(landed, 2 * bytes);
            ptx::tma_load_2d_pair(sa, &tm_a, bar, kb * kBlock, a_row);
            ptx::tma_load_2d_pair(sa + C::kABytes, &tm_b, bar, kb * kBlock, b_row);
            ptx::tma_load_2d_pair(scale, &tm_scale, bar, a_row, kb);
          } else {
            ptx::mbar_expect_tx(landed, bytes);
            ptx::tma_load_2d(sa, &tm_a, landed, kb * kBlock, a_row);
            ptx::tma_load_2d(sa + C::kABytes, &tm_b, landed, kb * kBlock, b_row);
            ptx::tma_load_2d(scale, &tm_scale, landed, a_row, kb);
          }
          ring.filled();
          if (++slot == C::kScaleSlots) slot = 0;
        }
      }
      if (!aborted(abort_flag) && !ring.wait_all_free(empty)) record_timeout(p.err, abort_flag);
      // Let loads in flight (both CTAs' count here) land before the end.
      if (aborted(abort_flag) && rank == 0) ring.drain(full);
    }
  } else if (warp == C::kEpilogueWarps + 1) {
    // ------------------------------------------------------------------ MMA issuer
    // The whole warp walks the loop and one lane issues, on descriptors that only
    // need an addition: this thread's instructions are the pipe's idle time (a
    // divergent lane building each descriptor took 900 cycles a block).
    if (rank == 0) {
      const uint32_t idesc = ptx::make_idesc_e4m3(kTileM * kCtas, kN);
      const uint64_t desc = kmajor_desc(ptx::smem_addr(smem), 128, 0);
      const bool issuer = ptx::elect_one();
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      for (int tile = first; tile < tiles && !aborted(abort_flag); tile += step) {
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!ptx::mbar_wait(&tmem_empty[buf], buf_phase ^ 1) ||
              !ptx::mbar_wait(&full[stage], phase)) {
            record_timeout(p.err, abort_flag);
            break;
          }
          ptx::tc_fence_after();
          if (issuer) {
            const uint64_t a_desc = desc + static_cast<uint32_t>(stage * (C::kOperandBytes / 16));
            const uint64_t b_desc = a_desc + C::kABytes / 16;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {  // 32 bytes further in the swizzle atom
              if constexpr (kCtas == 2) {
                ptx::mma_f8f6f4_pair(tmem + buf * kN, a_desc + 2 * ks, b_desc + 2 * ks, idesc,
                                     ks > 0);
              } else {
                ptx::mma_f8f6f4(tmem + buf * kN, a_desc + 2 * ks, b_desc + 2 * ks, idesc, ks > 0);
              }
            }
            if constexpr (kCtas == 2) {
              ptx::mma_commit_pair(&empty[stage]);
              ptx::mma_commit_pair(&tmem_full[buf]);
            } else {
              ptx::mma_commit(&empty[stage]);
              ptx::mma_commit(&tmem_full[buf]);
            }
          }
          __syncwarp();
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
          if (++buf == C::kBuffers) {
            buf = 0;
            buf_phase ^= 1;
          }
        }
      }
      if (aborted(abort_flag)) {
        if (issuer) {
          if constexpr (kCtas == 2) {
            ptx::mma_commit_leader(drain);
          } else {
            ptx::mma_commit(drain);
          }
        }
        ptx::mbar_wait(drain, 0, 200000000ull);
      }
    }
  } else if (warp < C::kEpilogueWarps) {
    // ------------------------------------------------------------------ epilogue
    if constexpr (C::kMoveRegs) ptx::raise_registers<C::kEpilogueRegs>();
    constexpr int kCols = C::kThreadCols;
    const int quarter = warp % 4;
    const int col = warp / 4 * kCols;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + col;
    const uint32_t empty_addr =  // in the CTA that issues the MMAs
        kCtas == 2 ? ptx::map_shared_rank(ptx::smem_addr(tmem_empty), 0) : 0;
    const uint32_t base = ptx::smem_addr(smem);
    const uint32_t scale0 = base + C::kScaleOffset + (quarter * 32 + lane) * 4;
    uint32_t scale_addr = scale0;
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = first; tile < tiles && !aborted(abort_flag); tile += step) {
      int tm, tn;
      band_order(tile, p.m_tiles, p.n_tiles, p.band, tm, tn);
      const int row0 = (tm * kCtas + static_cast<int>(rank)) * kTileM + quarter * 32;
      const int col0 = tn * kN + col;
      // Features of one thread lie in one 128-row block of b; each lane holds the
      // scale of one of the next 32 blocks of k.
      const float *b_scale =
          p.b_scales + static_cast<int64_t>(col0 < p.n ? col0 / kBlock : 0) * p.num_kb;
      float b_next = kb_begin + lane < kb_end ? __ldg(b_scale + kb_begin + lane) : 0.0f;
      float b_lane = 0.0f;
      float acc[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
      bool ok = true;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        const int in_chunk = (kb - kb_begin) & 31;
        if (in_chunk == 0) {
          b_lane = b_next;
          if (kb + 32 + lane < kb_end) b_next = __ldg(b_scale + kb + 32 + lane);
        }
        ok = !__any_sync(0xffffffffu, !ptx::mbar_wait(&tmem_full[buf], buf_phase));
        if (!ok) {
          if (lane == 0) record_timeout(p.err, abort_flag);
          break;
        }
        ptx::tc_fence_after();
        // The scales landed before the MMAs began, which this barrier follows.
        const float scale =
            ptx::ld_shared_f32(scale_addr) * __shfl_sync(0xffffffffu, b_lane, in_chunk);
        scale_addr += C::kScaleBytes;
        if (scale_addr == scale0 + C::kScaleSlots * C::kScaleBytes) scale_addr = scale0;
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += C::kAtOnce) {
          uint32_t v[C::kAtOnce / 32][32];
#pragma unroll
          for (int c = 0; c < C::kAtOnce / 32; ++c) {
            ptx::tmem_ld_32x32b_x32(t_row + buf * kN + c0 + c * 32, v[c]);
          }
          ptx::tmem_ld_wait();
          if (c0 + C::kAtOnce == kCols) {
            ptx::tc_fence_before();
            if constexpr (kCtas == 2) {
              ptx::warp_arrive_cluster(empty_addr + buf * 8);
            } else {
              ptx::warp_arrive(&tmem_empty[buf]);
            }
          }
#pragma unroll
          for (int e = 0; e < C::kAtOnce; ++e) {
            acc[c0 + e] = fmaf(scale, __uint_as_float(v[e / 32][e % 32]), acc[c0 + e]);
          }
        }
        if (++buf == C::kBuffers) {
          buf = 0;
          buf_phase ^= 1;
        }
      }
      if (!ok) break;
      if constexpr (kSplit) {
        // This share of the sums, column by column, over the spent ring.
        float *part = reinterpret_cast<float *>(smem) + quarter * 32 + lane;
#pragma unroll
        for (int e = 0; e < kCols; ++e) part[(col + e) * kTileM] = acc[e];
        continue;
      }
      // 32 columns at a time through this warp's buffer (64-byte rows, 16-byte
      // chunks swizzled as the tensor map expects, which spreads the banks).
      const uint32_t out = base + C::kOutOffset + warp * C::kOutBytes;
      const bool by_tma = p.n % 8 == 0;
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 32) {
        if (lane == 0) ptx::bulk_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float lo = acc[c0 + c * 8 + 2 * e], hi = acc[c0 + c * 8 + 2 * e + 1];
            w[e] = kBf16 ? ptx::pack_bf16x2(lo, hi) : ptx::pack_f16x2(lo, hi);
          }
          ptx::st_shared_v4(out + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4),
                            make_uint4(w[0], w[1], w[2], w[3]));
        }
        if (by_tma) {
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < p.m && col0 + c0 < p.n) {
            ptx::tma_store_2d_addr(&tm_y, out, col0 + c0, row0);
            ptx::bulk_commit();
          }
        } else {
          // Rows that are not whole 16-byte units: one row an instruction.
          __syncwarp();
          const int64_t n = col0 + c0 + lane;
          const int rows = min(32, static_cast<int>(min(p.m - row0, int64_t{32})));
          uint16_t *y = static_cast<uint16_t *>(p.y) + row0 * p.n + n;
          for (int r = 0; r < rows; ++r, y += p.n) {
            const uint32_t at = out + r * 64 + (((lane >> 3) ^ (r >> 1 & 3)) << 4) + (lane & 7) * 2;
            if (n < p.n) *y = ptx::ld_shared_u16(at);
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) ptx::bulk_wait_all();
  }

  ptx::tc_fence_before();
  __syncthreads();
  // Neither CTA leaves while the other's MMAs or arrivals may still reach it.
  if constexpr (kCtas == 2) ptx::cluster_sync();
  if constexpr (kSplit) {
    const int64_t row0 = static_cast<int64_t>(first / p.n_tiles) * kTileM;
    add_shares<kN, C::kEpilogueWarps * kWarp, kBf16>(
        ptx::smem_addr(smem), share, p.splits, static_cast<uint16_t *>(p.y) + row0 * p.n, p.n,
        p.m - row0, static_cast<int64_t>(first % p.n_tiles) * kN, p.n);
  }
  if (warp == C::kEpilogueWarps + 1) {
    ptx::tc_fence_after();
    if constexpr (kCtas == 2) {
      ptx::tmem_dealloc_pair(tmem, C::kTmemCols);
    } else {
      ptx::tmem_dealloc(tmem, C::kTmemCols);
    }
  }
}

// splits > 1: that many CTAs, a cluster, share a tile's blocks of k.
template <int kCtas, int kN, bool kBf16, bool kSplit = false>
int launch_tiles(Fp8Params p, cudaStream_t s, int splits = 1) {
  using C = TileCfg<kCtas, kN>;
  p.m_tiles = static_cast<int>((p.m + kCtas * kTileM - 1) / (kCtas * kTileM));
  p.n_tiles = static_cast<int>((p.n + kN - 1) / kN);
  // As many row blocks of a in a band as stay in L2 while b streams past.
  const int64_t fit = (int64_t{32} << 20) / (kCtas * kTileM * std::max<int64_t>(p.k, 1));
  p.band = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.m_tiles, fit)));
  if (kSplit) p.band = 1;  // row by row: a cluster finds its tile by a division
  p.splits = splits;
  p.err = device_error_word();
  if (p.err == nullptr) return record_cuda_error(cudaGetLastError());
  CUtensorMap tm_a, tm_b, tm_scale, tm_y;
  // A lone tile loads only the rows there are (whole groups of eight, the
  // swizzle's unit): the others' sums come from what is in shared memory and are
  // not stored. A full box on a matrix of a few rows loads slowly.
  p.a_rows = static_cast<int>(std::min<int64_t>(kTileM, (p.m + 7) / 8 * 8));
  if (int st = make_map(&tm_a, p.a, 1, p.k, p.m, kBlock, p.a_rows, true)) return st;
  if (int st = make_map(&tm_b, p.b, 1, p.k, p.n, kBlock, C::kBRows, true)) return st;
  if (int st = make_map(&tm_scale, p.a_scales, 4, p.m, p.num_kb, kTileM, 1, false, p.a_pitch)) {
    return st;
  }
  if (p.n % 8 == 0) {  // rows of whole 16-byte units; other results are stored element by element
    if (int st = make_map(&tm_y, p.y, 2, p.n, p.m, 32, 32, true)) return st;
  } else {
    tm_y = tm_a;
  }
  if (int st = allow_dynamic_smem<fp8_tile_kernel<kCtas, kN, kBf16, kSplit>>(C::kSmem)) return st;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(
      kSplit ? tiles * splits : std::min<int64_t>(tiles, sm_count() / kCtas) * kCtas));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kSplit ? splits : kCtas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  set_programmatic_dependency(attr[1]);
  cfg.attrs = attr;
  cfg.numAttrs = p.after_quantise ? 2 : 1;
  CFB_TRY_CUDA(cudaLaunchKernelEx(&cfg, fp8_tile_kernel<kCtas, kN, kBf16, kSplit>, tm_a, tm_b,
                                  tm_scale, tm_y, p));
  return check_launch();
}

template <typename T>
int matmul_fp8(const Fp8Params &p, cudaStream_t s) {
  if (p.m <= kStreamTokens) return launch_fp8_stream<T>(p, s);
  constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
  // The form with the least time by waves of tiles: a 128-block of k takes about
  // 1300 cycles of a pair's 256 x 256 tile, 780 of a 128 x 128 tile and 700 of a
  // 128 x 64 tile (measured at k = 4096).
  const int64_t sms = sm_count();
  auto cost = [&](int64_t tm, int64_t tn, int64_t slots, int64_t cycles) {
    const int64_t tiles = (p.m + tm - 1) / tm * ((p.n + tn - 1) / tn);
    return (tiles + slots - 1) / slots * cycles;
  };
  const int64_t pair = cost(256, 256, sms / 2, 1300), wide = cost(128, 128, sms, 780),
                narrow = cost(128, 64, sms, 700);
  // Few tiles: clusters share a tile's k, eight blocks at least to each CTA ([64,
  // 11008] x [4096, 11008] 27 -> 20 us; with four [64, 4096] x [1024, 4096] lost 1.6 of 12).
  const int splits = split_count((p.m + 127) / 128 * ((p.n + 63) / 64), p.num_kb, 8);
  if (splits > 1) return launch_tiles<1, 64, kBf16, true>(p, s, splits);
  if (pair <= wide && pair <= narrow) return launch_tiles<2, 256, kBf16>(p, s);
  return wide <= narrow ? launch_tiles<1, 128, kBf16>(p, s) : launch_tiles<1, 64, kBf16>(p, s);
}

int check_fp8_shape(int64_t m, int64_t k, int64_t n, int dtype) {
  if (m < 0 || k < 0 || n < 0) return CF_ERR_INVALID_ARGUMENT;
  if (dtype != CF_DTYPE_BF16 && dtype != CF_DTYPE_F16) return CF_ERR_UNSUPPORTED;
  if (m == 0 || n == 0) return CF_OK;
  if (k == 0 || k % 16 != 0) return CF_ERR_UNSUPPORTED;
  if (m > 0x7fffffffll - 256 || n > 0x7fffffffll - 256 || k > 0x7fffffffll - kBlock ||
      (m + 127) / 128 * ((n + 63) / 64) > 0x7fffffffll) {
    return CF_ERR_INVALID_ARGUMENT;  // tile counts and coordinates are 32-bit
  }
  return CF_OK;
}

Fp8Params fp8_params(const void *a, const float *a_scales, int64_t a_pitch, const uint8_t *b,
                     const float *b_scales, void *y, int64_t m, int64_t k, int64_t n) {
  Fp8Params p{};
  p.a = static_cast<const uint8_t *>(a);
  p.a_scales = a_scales;
  p.b = b;
  p.b_scales = b_scales;
  p.y = y;
  p.m = m;
  p.n = n;
  p.k = k;
  p.num_kb = static_cast<int>((k + kBlock - 1) / kBlock);
  p.a_pitch = a_pitch;
  return p;
}

int64_t fp8_scale_pitch(int64_t m) { return (m + 3) / 4 * 4; }

size_t fp8_code_bytes(int64_t m, int64_t k) {
  return (static_cast<size_t>(m) * static_cast<size_t>(k) + 255) & ~static_cast<size_t>(255);
}

}  // namespace
}  // namespace cfb

extern "C" {

int cf_quantize_fp8(const void *input, int dtype, uint8_t *codes, float *scales, int64_t rows,
                    int64_t cols, int block_rows, cf_stream_t stream) {
  if (rows < 0 || cols < 0) return CF_ERR_INVALID_ARGUMENT;
  if (dtype != CF_DTYPE_F32 && dtype != CF_DTYPE_BF16 && dtype != CF_DTYPE_F16) {
    return CF_ERR_UNSUPPORTED;
  }
  if (block_rows != 1 && block_rows != CF_FP8_BLOCK_SIZE) return CF_ERR_UNSUPPORTED;
  if (rows == 0 || cols == 0) return CF_OK;
  if (!input || !codes || !scales) return CF_ERR_INVALID_ARGUMENT;
  if (rows > (int64_t{1} << 40) / cols || cols > cfb::kQuantMaxCols) {
    return CF_ERR_INVALID_ARGUMENT;
  }
  return cfb::quantize_fp8_any(input, dtype, codes, scales, rows, cols, block_rows, 0,
                               reinterpret_cast<cudaStream_t>(stream));
}

int cf_matmul_fp8(const uint8_t *a_codes, const float *a_scales, int64_t a_scale_pitch,
                  const uint8_t *b_codes, const float *b_scales, void *y, int64_t m, int64_t k,
                  int64_t n, int dtype, cf_stream_t stream) {
  if (int st = cfb::check_fp8_shape(m, k, n, dtype)) return st;
  if (m == 0 || n == 0) return CF_OK;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !y) return CF_ERR_INVALID_ARGUMENT;
  if (a_scale_pitch < m) return CF_ERR_INVALID_ARGUMENT;
  if (a_scale_pitch % 4 != 0) return CF_ERR_UNSUPPORTED;
  if (!cfb::aligned_to(a_codes, 16) || !cfb::aligned_to(a_scales, 16) ||
      !cfb::aligned_to(b_codes, 16) || !cfb::aligned_to(y, 16)) {
    return CF_ERR_MISALIGNED;
  }
  const cfb::Fp8Params p =
      cfb::fp8_params(a_codes, a_scales, a_scale_pitch, b_codes, b_scales, y, m, k, n);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == CF_DTYPE_BF16 ? cfb::matmul_fp8<__nv_bfloat16>(p, s)
                                : cfb::matmul_fp8<__half>(p, s);
}

size_t cf_linear_fp8_workspace_bytes(int64_t m, int64_t k) {
  if (m <= 0 || k <= 0) return 0;
  const int64_t blocks = cfb::fp8_scale_pitch(m) * ((k + cfb::kBlock - 1) / cfb::kBlock);
  return cfb::fp8_code_bytes(m, k) + static_cast<size_t>(blocks) * sizeof(float);
}

int cf_linear_fp8(const void *x, const uint8_t *w_codes, const float *w_scales, void *y, int64_t m,
                  int64_t k, int64_t n, int dtype, void *workspace, size_t workspace_bytes,
                  cf_stream_t stream) {
  if (int st = cfb::check_fp8_shape(m, k, n, dtype)) return st;
  if (m == 0 || n == 0) return CF_OK;
  if (!x || !w_codes || !w_scales || !y || k > cfb::kQuantMaxCols) {
    return CF_ERR_INVALID_ARGUMENT;
  }
  if (!cfb::aligned_to(x, 16) || !cfb::aligned_to(w_codes, 16) || !cfb::aligned_to(y, 16)) {
    return CF_ERR_MISALIGNED;
  }
  if (workspace == nullptr || workspace_bytes < cf_linear_fp8_workspace_bytes(m, k)) {
    return CF_ERR_WORKSPACE;
  }
  if (!cfb::aligned_to(workspace, 16)) return CF_ERR_MISALIGNED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  uint8_t *codes = static_cast<uint8_t *>(workspace);
  float *scales = reinterpret_cast<float *>(codes + cfb::fp8_code_bytes(m, k));
  const int64_t pitch = cfb::fp8_scale_pitch(m);
  if (int st = cfb::quantize_fp8_any(x, dtype, codes, scales, m, k, 1, pitch, s)) return st;
  cfb::Fp8Params p = cfb::fp8_params(codes, scales, pitch, w_codes, w_scales, y, m, k, n);
  p.after_quantise = true;
  return dtype == CF_DTYPE_BF16 ? cfb::matmul_fp8<__nv_bfloat16>(p, s)
                                : cfb::matmul_fp8<__half>(p, s);
}

}  // extern "C"
