// The gate and up projections of a feed-forward block with their activation and
// product in one kernel, and the backward pass, for sm_100a (f16 and bf16):
//
//   g = x Wg^T,  u = x Wu^T,  y = act(g) u          x [m, k], Wg, Wu [n, k]
//   dg = dy u act'(g),  du = dy act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
// with act(v) = v s(v), s = 1 / (1 + exp(-v)) for SiLU and 1 / (1 + exp(-2 z)),
// z = sqrt(2/pi) (v + 0.044715 v^3), for the tanh form of GELU (v (1 + tanh z) / 2).
//
// Sums are fp32; y, dx, dWg and dWu are each rounded once. For the backward pass
// the forward one keeps g and u in fp32 (8 bytes an element; kept in 16 bits
// their roundings would nearly double the error of dg and du, recomputing them
// would add a third to the products of a step). dg and du are rounded to the
// operands' type, which the tensor core's 16-bit products need.
//
// Tensor-bound: 4 m n k forward, 8 m n k backward. One tile kernel serves the
// three products, with K-major or MN-major operands as they lie in memory: CTA
// pairs, 256 x 256 tiles, two accumulators in TMEM so that a tile's end hides
// behind the next one's products. [4096, 4096] x 2 x [11008, 4096] bf16: forward
// 427 us (1.73 PFLOP/s), with g and u kept 466 us, backward 1.08 ms (1.37), of
// which dg and du 0.1 ms; in a loop the power limit takes 15 % off that. Up to 8
// tokens the forward pass is bound by the weights' bytes and streams them (4
// tokens: 31 us, 5.8 TB/s).
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

// ---------------------------------------------------------------- activations

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// The sigmoid factor of the activation.
__device__ __forceinline__ float gate_sigmoid(float v, int act) {
  const float z = act == CF_ACT_SILU ? v : 2.0f * kGeluC * v * fmaf(kGeluA * v, v, 1.0f);
  return __fdividef(1.0f, 1.0f + __expf(-z));
}

// Activation and its derivative s + v s (1 - s) z', z' the factor's slope.
__device__ __forceinline__ void gate_slope(float v, int act, float &value, float &slope) {
  const float s = gate_sigmoid(v, act);
  value = v * s;
  const float zp = act == CF_ACT_SILU ? 1.0f : 2.0f * kGeluC * fmaf(3.0f * kGeluA * v, v, 1.0f);
  const float tail = value * (1.0f - s);  // 0 where the factor has saturated, whatever zp is
  slope = tail == 0.0f ? s : fmaf(tail, zp, s);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return kBf16 ? ptx::pack_bf16x2(lo, hi) : ptx::pack_f16x2(lo, hi);
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
  }
}

// ---------------------------------------------------------------- tiles

struct GatedParams {
  int64_t m, n, k;
  int num_kb;      // 64-blocks of the contracted dimension
  int split_kb;    // kInput: blocks of the first of its two products
  int m_tiles, n_tiles, band;
  int matrices;    // kWeights: 1 or 2 gradients
  int splits;      // CTAs that share a tile's contracted blocks
  int a_rows;      // rows of x (or dg, du) in a stage, fewer than a tile's where m ends before
  int act;
  bool save;       // kForward: keep g and u
  const void *x, *w_gate, *w_up;
  void *y;
  unsigned *err;
};

// kForward: A = x, B = 128 rows of Wg and the same 128 of Wu, both K-major; the
//   accumulator's columns are 128 gates and their 128 ups, so a thread (a token)
//   has both.
// kInput: A = dg, then du (K-major), B = Wg, then Wu (contracted rows, MN-major).
// kWeights: A = dg or du, B = x, both MN-major (contracted over the tokens).
enum GatedMode { kForward, kInput, kWeights };

constexpr int kTileRows = 128;     // of D in one CTA
constexpr int kTileCols = 256;     // TMEM columns of one accumulator
constexpr int kDepth = 64;         // 16-bit elements of a 128-byte swizzle row
constexpr int kGatedThreads = 384; // warps 0-7 epilogue, 8 producer, 9 MMA, 10-11 idle
constexpr int kEpilogueBytes = 32 * 128;  // a warp's 32 rows of 128 bytes on their way out

// kCtas = 2: CTA pairs of 256 rows, each CTA staging 128 rows of A and of B
// (forward: one of them the gate's, the other the up's).
template <int kCtas>
struct GatedCfg {
  static constexpr int kABytes = kTileRows * kDepth * 2;
  static constexpr int kBRows = kTileCols / kCtas;
  static constexpr int kStageBytes = kABytes + kBRows * kDepth * 2;
  static constexpr int kStages = 196608 / kStageBytes;
  static constexpr int kOutOffset = kStages * kStageBytes;
  static constexpr int kBarOffset = kOutOffset + 8 * kEpilogueBytes;
  static constexpr size_t kSmem = 1024 + kBarOffset + 256;
  static_assert(kSmem <= 232448, "227 KB of shared memory");
};

struct GatedMaps {
  CUtensorMap a[2], b[2], out[2], save[2];
};

// kSplit: the CTAs of a cluster share a tile's contracted blocks and add their
// sums through distributed shared memory (few tokens leave too few tiles of dx).
template <int kMode, int kCtas, bool kBf16, bool kSplit>
__global__ void __launch_bounds__(kGatedThreads, 1)
    gated_tile_kernel(const __grid_constant__ GatedMaps maps, const GatedParams p) {
  static_assert(!kSplit || (kMode == kInput && kCtas == 1), "the split product");
  using C = GatedCfg<kCtas>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::kBarOffset);
  uint64_t *empty = full + C::kStages;
  uint64_t *tmem_full = empty + C::kStages;  // [2]
  uint64_t *tmem_empty = tmem_full + 2;      // [2]
  uint64_t *drain = tmem_empty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  int *abort_flag = reinterpret_cast<int *>(tmem_slot + 1);
  const int warp = threadIdx.x / kWarp;
  const int lane = threadIdx.x % kWarp;
  const int rank = kCtas == 2 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int per_matrix = p.m_tiles * p.n_tiles;
  const int tiles = per_matrix * (kMode == kWeights ? p.matrices : 1);
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
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&tmem_full[i], 1);
      ptx::mbar_init(&tmem_empty[i], kCtas * 8);
    }
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 9) {
    if constexpr (kCtas == 2) {
      ptx::tmem_alloc_pair(tmem_slot, 512);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, 512);
      ptx::tmem_relinquish();
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (kCtas == 2) ptx::cluster_sync();  // both CTAs' barriers are ready
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 8) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      StageRing<C::kStages> ring;
      for (int tile = first; tile < tiles && !aborted(abort_flag); tile += step) {
        const int which = kMode == kWeights ? tile / per_matrix : 0;
        int tm, tn;
        band_order(tile - which * per_matrix, p.m_tiles, p.n_tiles, p.band, tm, tn);
        const int row = (tm * kCtas + rank) * kTileRows;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!ring.wait_free(empty)) {
            record_timeout(p.err, abort_flag);
            break;
          }
          uint64_t *const landed = &full[ring.stage];
          uint8_t *sa = smem + ring.stage * C::kStageBytes;
          uint8_t *sb = sa + C::kABytes;
          // The even CTA's barrier counts both CTAs' bytes.
          const uint32_t bar = kCtas == 2 ? ptx::map_shared_rank(ptx::smem_addr(landed), 0)
                                          : ptx::smem_addr(landed);
          const uint32_t bytes =
              kMode == kWeights ? C::kStageBytes : C::kStageBytes - (kTileRows - p.a_rows) * 128;
          if (rank == 0) ptx::mbar_expect_tx(landed, kCtas * bytes);
          auto load = [&](uint8_t *dst, const CUtensorMap *map, int c0, int c1) {
            if constexpr (kCtas == 2) {
              ptx::tma_load_2d_pair(dst, map, bar, c0, c1);
            } else {
              ptx::tma_load_2d(dst, map, landed, c0, c1);
            }
          };
          // MN-major: chunks of 64 columns (one swizzle row) x 64 contracted rows.
          constexpr int kChunkBytes = kDepth * 128;
          if constexpr (kMode == kForward) {
            load(sa, &maps.a[0], kb * kDepth, row);
            if constexpr (kCtas == 2) {
              load(sb, &maps.b[rank], kb * kDepth, tn * 128);
            } else {
              load(sb, &maps.b[0], kb * kDepth, tn * 128);
              load(sb + 128 * 128, &maps.b[1], kb * kDepth, tn * 128);
            }
          } else {
            const int col = tn * kTileCols + rank * C::kBRows;
            if constexpr (kMode == kInput) {
              const int second = kb >= p.split_kb;
              const int at = (kb - (second ? p.split_kb : 0)) * kDepth;
              load(sa, &maps.a[second], at, row);
#pragma unroll
              for (int c = 0; c < C::kBRows / 64; ++c) {
                load(sb + c * kChunkBytes, &maps.b[second], col + c * 64, at);
              }
            } else {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                load(sa + c * kChunkBytes, &maps.a[which], row + c * 64, kb * kDepth);
              }
#pragma unroll
              for (int c = 0; c < C::kBRows / 64; ++c) {
                load(sb + c * kChunkBytes, &maps.b[0], col + c * 64, kb * kDepth);
              }
            }
          }
          ring.filled();
        }
      }
      if (!aborted(abort_flag) && !ring.wait_all_free(empty)) record_timeout(p.err, abort_flag);
      // Let loads in flight (both CTAs' count here) land before the end.
      if (aborted(abort_flag) && rank == 0) ring.drain(full);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA issuer
    // The whole warp walks the loop, one lane issues; descriptors advance by
    // addition (a divergent lane that builds each one starves the pipe).
    if (rank == 0) {
      constexpr bool kAMn = kMode == kWeights, kBMn = kMode != kForward;
      const uint32_t idesc =
          ptx::make_idesc_f16(kBf16, kTileRows * kCtas, kTileCols, kAMn, kBMn);
      const uint32_t base = ptx::smem_addr(smem);
      const uint64_t a0 =
          kAMn ? mnmajor_desc(base, 128, kDepth * 128, 0) : kmajor_desc(base, 128, 0);
      const uint64_t b0 = kBMn ? mnmajor_desc(base + C::kABytes, 128, kDepth * 128, 0)
                               : kmajor_desc(base + C::kABytes, 128, 0);
      // 16 contracted elements: 32 bytes of a row, or 16 rows of 128 bytes.
      constexpr uint32_t kAStep = kAMn ? 128 : 2, kBStep = kBMn ? 128 : 2;
      const bool issuer = ptx::elect_one();
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      for (int tile = first; tile < tiles && !aborted(abort_flag); tile += step) {
        bool ok = ptx::mbar_wait(&tmem_empty[buf], buf_phase ^ 1);
        ptx::tc_fence_after();
        const uint32_t d = tmem + buf * kTileCols;
        for (int kb = kb_begin; ok && kb < kb_end; ++kb) {
          ok = ptx::mbar_wait(&full[stage], phase);
          if (!ok) break;
          ptx::tc_fence_after();
          if (issuer) {
            const uint32_t off = static_cast<uint32_t>(stage * (C::kStageBytes / 16));
            const uint64_t a = a0 + off, b = b0 + off;
#pragma unroll
            for (int ks = 0; ks < kDepth / 16; ++ks) {
              if constexpr (kCtas == 2) {
                ptx::mma_f16_pair(d, a + ks * kAStep, b + ks * kBStep, idesc,
                                  kb > kb_begin || ks > 0);
              } else {
                ptx::mma_f16(d, a + ks * kAStep, b + ks * kBStep, idesc, kb > kb_begin || ks > 0);
              }
            }
            if constexpr (kCtas == 2) {
              ptx::mma_commit_pair(&empty[stage]);
            } else {
              ptx::mma_commit(&empty[stage]);
            }
          }
          __syncwarp();
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) {
          record_timeout(p.err, abort_flag);
          break;
        }
        if (issuer) {
          if constexpr (kCtas == 2) {
            ptx::mma_commit_pair(&tmem_full[buf]);
          } else {
            ptx::mma_commit(&tmem_full[buf]);
          }
        }
        __syncwarp();
        buf ^= 1;
        if (buf == 0) buf_phase ^= 1;
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
  } else if (warp < 8) {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp % 4, half = warp / 4;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t empty_addr =
        kCtas == 2 ? ptx::map_shared_rank(ptx::smem_addr(tmem_empty), 0) : 0;
    const uint32_t out = ptx::smem_addr(smem) + C::kOutOffset + warp * kEpilogueBytes;
    auto release = [&](int buf) {
      ptx::tc_fence_before();
      if constexpr (kCtas == 2) {
        ptx::warp_arrive_cluster(empty_addr + buf * 8);
      } else {
        ptx::warp_arrive(&tmem_empty[buf]);
      }
    };
    // 32 rows x 32 results of this warp, through its buffer and TMA (16-byte
    // chunks swizzled as the tensor map expects, which spreads the banks).
    auto store16 = [&](const uint32_t (&w)[16], const CUtensorMap *map, int col, int row,
                       int64_t cols, int64_t rows) {
      if (lane == 0) ptx::bulk_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        ptx::st_shared_v4(out + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4),
                          make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && row < rows && col < cols) {
        ptx::tma_store_2d_addr(map, out, col, row);
        ptx::bulk_commit();
      }
    };
    auto store32 = [&](const uint32_t (&v)[32], const CUtensorMap *map, int col, int row) {
      if (lane == 0) ptx::bulk_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        ptx::st_shared_v4(out + lane * 128 + ((c ^ (lane & 7)) << 4),
                          make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]));
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && row < p.m && col < p.n) {
        ptx::tma_store_2d_addr(map, out, col, row);
        ptx::bulk_commit();
      }
    };
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = first; tile < tiles && !aborted(abort_flag); tile += step) {
      const int which = kMode == kWeights ? tile / per_matrix : 0;
      int tm, tn;
      band_order(tile - which * per_matrix, p.m_tiles, p.n_tiles, p.band, tm, tn);
      const int row = (tm * kCtas + rank) * kTileRows + quarter * 32;
      if (__any_sync(0xffffffffu, !ptx::mbar_wait(&tmem_full[buf], buf_phase))) {
        if (lane == 0) record_timeout(p.err, abort_flag);
        break;
      }
      ptx::tc_fence_after();
      const uint32_t acc = t_row + buf * kTileCols;
      if constexpr (kMode == kForward) {
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const int at = half * 64 + c * 32;
          uint32_t g[32], u[32], w[16];
          ptx::tmem_ld_32x32b_x32(acc + at, g);
          ptx::tmem_ld_32x32b_x32(acc + 128 + at, u);
          ptx::tmem_ld_wait();
          if (c == 1) release(buf);
          const int col = tn * 128 + at;
          if (p.save) {
            store32(g, &maps.save[0], col, row);
            store32(u, &maps.save[1], col, row);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float g0 = __uint_as_float(g[2 * e]), g1 = __uint_as_float(g[2 * e + 1]);
            w[e] = pack2<kBf16>(g0 * gate_sigmoid(g0, p.act) * __uint_as_float(u[2 * e]),
                                g1 * gate_sigmoid(g1, p.act) * __uint_as_float(u[2 * e + 1]));
          }
          store16(w, &maps.out[0], col, row, p.n, p.m);
        }
      } else {
        const int64_t rows = kMode == kInput ? p.m : p.n;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int at = half * 128 + c * 32;
          uint32_t v[32], w[16];
          ptx::tmem_ld_32x32b_x32(acc + at, v);
          ptx::tmem_ld_wait();
          if (c == 3) release(buf);
          if constexpr (kSplit) {
            // This share of the sums, column by column, over the spent ring.
            float *part = reinterpret_cast<float *>(smem) + quarter * 32 + lane;
#pragma unroll
            for (int e = 0; e < 32; ++e) part[(at + e) * kTileRows] = __uint_as_float(v[e]);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            w[e] = pack2<kBf16>(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
          }
          store16(w, &maps.out[which], tn * kTileCols + at, row, p.k, rows);
        }
      }
      buf ^= 1;
      if (buf == 0) buf_phase ^= 1;
    }
    if (lane == 0) ptx::bulk_wait_all();
  }

  ptx::tc_fence_before();
  __syncthreads();
  // Neither CTA leaves while the other's MMAs or arrivals may still reach it.
  if constexpr (kCtas == 2) ptx::cluster_sync();
  if constexpr (kSplit) {
    const int64_t row0 = static_cast<int64_t>(first / p.n_tiles) * kTileRows;
    add_shares<kTileCols, 8 * kWarp, kBf16>(
        ptx::smem_addr(smem), share, p.splits, static_cast<uint16_t *>(p.y) + row0 * p.k, p.k,
        p.m - row0, static_cast<int64_t>(first % p.n_tiles) * kTileCols, p.k);
  }
  if (warp == 9) {
    ptx::tc_fence_after();
    if constexpr (kCtas == 2) {
      ptx::tmem_dealloc_pair(tmem, 512);
    } else {
      ptx::tmem_dealloc(tmem, 512);
    }
  }
}

template <int kMode, int kCtas, bool kBf16, bool kSplit = false>
int launch_tiles(const GatedMaps &maps, GatedParams p, int64_t rows, int64_t cols, int tile_cols,
                 cudaStream_t s) {
  using C = GatedCfg<kCtas>;
  p.m_tiles = static_cast<int>((rows + kCtas * kTileRows - 1) / (kCtas * kTileRows));
  p.n_tiles = static_cast<int>((cols + tile_cols - 1) / tile_cols);
  // As many row blocks of the A operand in a band as stay in L2 while B streams past.
  const int64_t fit = (int64_t{32} << 20) / (int64_t{kCtas} * kTileRows * p.num_kb * kDepth * 2);
  p.band = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.m_tiles, fit)));
  if (kSplit) p.band = 1;  // row by row: a cluster finds its tile by a division
  p.err = device_error_word();
  if (p.err == nullptr) return record_cuda_error(cudaGetLastError());
  if (int st = allow_dynamic_smem<gated_tile_kernel<kMode, kCtas, kBf16, kSplit>>(C::kSmem)) {
    return st;
  }
  const int64_t tiles =
      int64_t{p.m_tiles} * p.n_tiles * (kMode == kWeights ? p.matrices : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(
      kSplit ? tiles * p.splits : std::min<int64_t>(tiles, sm_count() / kCtas) * kCtas));
  cfg.blockDim = dim3(kGatedThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kSplit ? p.splits : kCtas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CFB_TRY_CUDA(cudaLaunchKernelEx(&cfg, gated_tile_kernel<kMode, kCtas, kBf16, kSplit>, maps, p));
  return check_launch();
}

// ---------------------------------------------------------------- few tokens

// The streaming kernel with m16n8k16: a block is 64 elements of k, a stage
// four blocks of Wg (warps 0-3) and the same of Wu (warps 4-7).
constexpr int kStreamBlocks = kStreamWarps / 2;

template <bool kBf16>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

template <bool kBf16>
struct GatedStreamOp {
  static constexpr int kMatrices = 2, kBlocks = kStreamBlocks, kBlockElems = kDepth;
  static constexpr int kScaleBytes = 0;
  struct Weights {};

  StreamMap w[2], less[2], tokens;
  GatedParams p;
  float *gate, *up;  // g and u for the backward pass, or null
  unsigned *err;
  StreamTiles tiles;
  int steps, whole_steps, blocks, token_rows, scale_bytes;

  __device__ __forceinline__ void load_scales(uint8_t *, uint64_t *, int) const {}
  __device__ __forceinline__ void fetch(Weights &, int, int, int) const {}

  __device__ __forceinline__ void multiply(const StreamRows &r, const uint4 (&x)[2],
                                           const float (&)[2], const Weights &, int, int,
                                           float (&acc)[4]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mma_16x8x16<kBf16>(acc, r.w[0][h].x, r.w[1][h].x, r.w[0][h].y, r.w[1][h].y, x[h].x, x[h].y);
      mma_16x8x16<kBf16>(acc, r.w[0][h].z, r.w[1][h].z, r.w[0][h].w, r.w[1][h].w, x[h].z, x[h].w);
    }
  }

  __device__ __forceinline__ void store(int feature, int count, const float *red) const {
    if (threadIdx.x >= kStreamTokens * kStreamFeatures) return;
    const int m = threadIdx.x / kStreamFeatures, f = threadIdx.x % kStreamFeatures;
    const int64_t n = int64_t{feature} + f;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < kStreamBlocks; ++w) {
      g += red[(w * kStreamTokens + m) * kStreamRedRow + f];
      u += red[((w + kStreamBlocks) * kStreamTokens + m) * kStreamRedRow + f];
    }
    if (m < p.m && f < count && n < p.n) {
      const int64_t at = m * p.n + n;
      const float v = g * gate_sigmoid(g, p.act) * u;
      static_cast<uint16_t *>(p.y)[at] = static_cast<uint16_t>(pack2<kBf16>(v, 0.0f));
      if (gate != nullptr) {
        gate[at] = g;
        up[at] = u;
      }
    }
  }
};

template <bool kBf16>
int launch_gated_stream(const GatedParams &p, float *gate, float *up, cudaStream_t s) {
  GatedStreamOp<kBf16> op;
  op.p = p;
  op.gate = gate;
  op.up = up;
  op.err = device_error_word();
  if (op.err == nullptr) return record_cuda_error(cudaGetLastError());
  op.tiles = stream_tiles(p.n);
  op.blocks = p.num_kb;
  op.steps = (p.num_kb + kStreamBlocks - 1) / kStreamBlocks;
  op.token_rows = static_cast<int>(p.m);
  op.scale_bytes = 0;
  op.whole_steps = stream_whole_steps(p.k * 2, kStreamBlocks);
  auto map = [&](StreamMap &to, const void *base, int64_t n, int rows) {
    return to.make(base, 2, p.k, n, rows, kStreamBlocks, op.whole_steps);
  };
  if (int st = map(op.tokens, p.x, p.m, op.token_rows)) return st;
  const void *w[2] = {p.w_gate, p.w_up};
  for (int i = 0; i < 2; ++i) {
    if (int st = map(op.w[i], w[i], p.n, op.tiles.rows)) return st;
    if (int st = map(op.less[i], w[i], p.n, std::max(1, op.tiles.rows - 1))) return st;
  }
  return launch_stream(op, false, s);
}

// ---------------------------------------------------------------- dg and du

// Elementwise and HBM-bound: reads dy, g and u, writes dg and du (14 bytes an
// element). `count` is a multiple of 8; the pointers are 16-byte aligned.
template <bool kBf16>
__global__ void __launch_bounds__(256)
    gated_slopes_kernel(const uint4 *dy, const float4 *g, const float4 *u, uint4 *dg, uint4 *du,
                        int64_t count, int act) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i * 8 >= count) return;
  const uint4 d = __ldcs(dy + i);
  const float4 g0 = __ldcs(g + 2 * i), g1 = __ldcs(g + 2 * i + 1);
  const float4 u0 = __ldcs(u + 2 * i), u1 = __ldcs(u + 2 * i + 1);
  const uint32_t dw[4] = {d.x, d.y, d.z, d.w};
  const float gv[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
  const float uv[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
  uint32_t og[4], ou[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v = unpack2<kBf16>(dw[e]);
    float a0, s0, a1, s1;
    gate_slope(gv[2 * e], act, a0, s0);
    gate_slope(gv[2 * e + 1], act, a1, s1);
    og[e] = pack2<kBf16>(v.x * uv[2 * e] * s0, v.y * uv[2 * e + 1] * s1);
    ou[e] = pack2<kBf16>(v.x * a0, v.y * a1);
  }
  dg[i] = make_uint4(og[0], og[1], og[2], og[3]);
  du[i] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
}

// ---------------------------------------------------------------- host

// A lone tile loads only the rows there are (whole groups of eight, the swizzle's
// unit): the others' sums come from what is in shared memory and are not stored. A
// full box on a matrix of a few rows loads slowly.
int tile_rows(int64_t m) {
  return static_cast<int>(std::min<int64_t>(kTileRows, (m + 7) / 8 * 8));
}

template <bool kBf16>
int forward(GatedParams p, float *g, float *u, cudaStream_t s) {
  if (p.m <= kStreamTokens) return launch_gated_stream<kBf16>(p, g, u, s);
  GatedMaps maps;
  const void *w[2] = {p.w_gate, p.w_up};
  float *save[2] = {g, u};
  p.a_rows = tile_rows(p.m);
  if (int st = make_map(&maps.a[0], p.x, 2, p.k, p.m, kDepth, p.a_rows, true)) return st;
  maps.a[1] = maps.a[0];
  for (int i = 0; i < 2; ++i) {
    if (int st = make_map(&maps.b[i], w[i], 2, p.k, p.n, kDepth, 128, true)) return st;
  }
  if (int st = make_map(&maps.out[0], p.y, 2, p.n, p.m, 32, 32, true)) return st;
  maps.out[1] = maps.save[0] = maps.save[1] = maps.out[0];
  if (p.save) {
    for (int i = 0; i < 2; ++i) {
      if (int st = make_map(&maps.save[i], save[i], 4, p.n, p.m, 32, 32, true)) return st;
    }
  }
  // Pairs of CTAs, 256 tokens each, where their tiles keep the GPU as full.
  const int64_t sms = sm_count(), n_tiles = (p.n + 127) / 128;
  const int64_t pairs = (p.m + 255) / 256 * n_tiles, singles = (p.m + 127) / 128 * n_tiles;
  const bool pair =
      p.m > kTileRows && (pairs + sms / 2 - 1) / (sms / 2) <= (singles + sms - 1) / sms;
  return pair ? launch_tiles<kForward, 2, kBf16>(maps, p, p.m, p.n, 128, s)
              : launch_tiles<kForward, 1, kBf16>(maps, p, p.m, p.n, 128, s);
}

template <bool kBf16>
int backward(GatedParams p, const void *dy, const float *g, const float *u, void *dg, void *du,
             void *dx, void *dw_gate, void *dw_up, cudaStream_t s) {
  const int64_t count = p.m * p.n;
  const int64_t grid = (count / 8 + 255) / 256;
  gated_slopes_kernel<kBf16><<<static_cast<unsigned>(grid), 256, 0, s>>>(
      static_cast<const uint4 *>(dy), reinterpret_cast<const float4 *>(g),
      reinterpret_cast<const float4 *>(u), static_cast<uint4 *>(dg), static_cast<uint4 *>(du),
      count, p.act);
  if (int st = check_launch()) return st;
  const void *d[2] = {dg, du}, *w[2] = {p.w_gate, p.w_up};
  GatedMaps maps;
  if (dx != nullptr) {
    for (int i = 0; i < 2; ++i) {
      if (int st = make_map(&maps.a[i], d[i], 2, p.n, p.m, kDepth, tile_rows(p.m), true)) {
        return st;
      }
      if (int st = make_map(&maps.b[i], w[i], 2, p.k, p.n, 64, kDepth, true)) return st;
    }
    if (int st = make_map(&maps.out[0], dx, 2, p.k, p.m, 32, 32, true)) return st;
    maps.out[1] = maps.save[0] = maps.save[1] = maps.out[0];
    p.split_kb = static_cast<int>((p.n + kDepth - 1) / kDepth);
    p.num_kb = 2 * p.split_kb;
    p.a_rows = tile_rows(p.m);
    p.y = dx;
    p.splits = split_count((p.m + 127) / 128 * ((p.k + kTileCols - 1) / kTileCols), p.num_kb, 16);
    const int st =
        p.splits > 1
            ? launch_tiles<kInput, 1, kBf16, true>(maps, p, p.m, p.k, kTileCols, s)
            : launch_tiles<kInput, 2, kBf16>(maps, p, p.m, p.k, kTileCols, s);
    if (st != CF_OK) return st;
  }
  void *dw[2] = {dw_gate, dw_up};
  p.matrices = 0;
  for (int i = 0; i < 2; ++i) {
    if (dw[i] == nullptr) continue;
    if (int st = make_map(&maps.a[p.matrices], d[i], 2, p.n, p.m, 64, kDepth, true)) return st;
    if (int st = make_map(&maps.out[p.matrices], dw[i], 2, p.k, p.n, 32, 32, true)) return st;
    ++p.matrices;
  }
  if (p.matrices == 0) return CF_OK;
  if (p.matrices == 1) {
    maps.a[1] = maps.a[0];
    maps.out[1] = maps.out[0];
  }
  if (int st = make_map(&maps.b[0], p.x, 2, p.k, p.m, 64, kDepth, true)) return st;
  maps.b[1] = maps.b[0];
  maps.save[0] = maps.save[1] = maps.out[0];
  p.num_kb = static_cast<int>((p.m + kDepth - 1) / kDepth);
  return launch_tiles<kWeights, 2, kBf16>(maps, p, p.n, p.k, kTileCols, s);
}

int check_gated(int64_t m, int64_t k, int64_t n, int act, int dtype) {
  if (m < 0 || k < 0 || n < 0) return CF_ERR_INVALID_ARGUMENT;
  if (act != CF_ACT_SILU && act != CF_ACT_GELU) return CF_ERR_INVALID_ARGUMENT;
  if (dtype != CF_DTYPE_BF16 && dtype != CF_DTYPE_F16) return CF_ERR_UNSUPPORTED;
  if (m == 0 || n == 0) return CF_OK;
  if (k == 0 || k % 8 != 0 || n % 8 != 0) return CF_ERR_UNSUPPORTED;
  // Tile counts and coordinates are 32-bit.
  const int64_t top = 0x7fffffffll - 512;
  if (m > top || n > top || k > top || (m + 127) / 128 * ((n + 127) / 128) > top ||
      (m + 127) / 128 * ((k + 127) / 128) > top || (n + 127) / 128 * ((k + 127) / 128) > top ||
      m * n / 8 > top * 256) {
    return CF_ERR_INVALID_ARGUMENT;
  }
  return CF_OK;
}

bool aligned_all(std::initializer_list<const void *> pointers) {
  for (const void *p : pointers) {
    if (!aligned_to(p, 16)) return false;  // a null pointer is aligned
  }
  return true;
}

GatedParams gated_params(const void *x, const void *w_gate, const void *w_up, int64_t m, int64_t k,
                         int64_t n, int act) {
  GatedParams p{};
  p.x = x;
  p.w_gate = w_gate;
  p.w_up = w_up;
  p.m = m;
  p.n = n;
  p.k = k;
  p.num_kb = static_cast<int>((k + kDepth - 1) / kDepth);
  p.act = act;
  return p;
}

size_t gated_plane_bytes(int64_t m, int64_t n) {
  return (static_cast<size_t>(m) * static_cast<size_t>(n) * 2 + 255) & ~static_cast<size_t>(255);
}

}  // namespace
}  // namespace cfb

extern "C" {

int cf_gated_linear(const void *x, const void *w_gate, const void *w_up, void *y, float *gate,
                    float *up, int64_t m, int64_t k, int64_t n, int activation, int dtype,
                    cf_stream_t stream) {
  if (int st = cfb::check_gated(m, k, n, activation, dtype)) return st;
  if (m == 0 || n == 0) return CF_OK;
  if (!x || !w_gate || !w_up || !y || (gate == nullptr) != (up == nullptr)) {
    return CF_ERR_INVALID_ARGUMENT;
  }
  if (!cfb::aligned_all({x, w_gate, w_up, y, gate, up})) return CF_ERR_MISALIGNED;
  cfb::GatedParams p = cfb::gated_params(x, w_gate, w_up, m, k, n, activation);
  p.y = y;
  p.save = gate != nullptr;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == CF_DTYPE_BF16 ? cfb::forward<true>(p, gate, up, s)
                                : cfb::forward<false>(p, gate, up, s);
}

size_t cf_gated_linear_backward_workspace_bytes(int64_t m, int64_t n) {
  return m <= 0 || n <= 0 ? 0 : 2 * cfb::gated_plane_bytes(m, n);
}

int cf_gated_linear_backward(const void *dy, const void *x, const void *w_gate, const void *w_up,
                             const float *gate, const float *up, void *dx, void *dw_gate,
                             void *dw_up, int64_t m, int64_t k, int64_t n, int activation,
                             int dtype, void *workspace, size_t workspace_bytes,
                             cf_stream_t stream) {
  if (int st = cfb::check_gated(m, k, n, activation, dtype)) return st;
  if (m == 0 || n == 0) return CF_OK;
  if (!dy || !x || !w_gate || !w_up || !gate || !up) return CF_ERR_INVALID_ARGUMENT;
  if (workspace == nullptr ||
      workspace_bytes < cf_gated_linear_backward_workspace_bytes(m, n)) {
    return CF_ERR_WORKSPACE;
  }
  if (!cfb::aligned_all({dy, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, workspace})) {
    return CF_ERR_MISALIGNED;
  }
  const cfb::GatedParams p = cfb::gated_params(x, w_gate, w_up, m, k, n, activation);
  void *dg = workspace;
  void *du = static_cast<char *>(workspace) + cfb::gated_plane_bytes(m, n);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == CF_DTYPE_BF16
             ? cfb::backward<true>(p, dy, gate, up, dg, du, dx, dw_gate, dw_up, s)
             : cfb::backward<false>(p, dy, gate, up, dg, du, dx, dw_gate, dw_up, s);
}

}  // extern "C"
