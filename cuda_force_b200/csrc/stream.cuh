// A product with up to eight tokens: bound by reading the weights once. Persistent CTAs
// walk over tiles of up to 16 output features; a producer warp streams the tiles' rows
// and the tokens, eight blocks of 128 bytes of k a stage, through a ring in shared memory
// by TMA. Each of eight consumer warps multiplies one block of the features with all
// tokens on the warp-wide MMA (features as M, tokens as N): at these shapes the tensor
// core's rate does not matter. The warps' sums of a tile meet in shared memory. Two CTAs
// on an SM, so that one's tile ends hide behind the other's loads.
//
// [8, 8192] x 2 x [28672, 8192] bf16: 138 us, 6.8 TB/s (a copy for each block and tokens
// loaded by their consumers, a step ahead: 190; the same with full tiles and a last round
// for some CTAs: 191). [8, 8192] x [28672, 8192] in e4m3, with the tokens' quantisation:
// 45 us (49). One CTA on an SM with twice the stages was a fifth slower.
//
// A lane's fragment words of a feature are 32 consecutive bytes of the block: any
// order of the contracted elements will do as long as both operands use it.
#pragma once

#include "cf_common.cuh"
#include "gemm_common.cuh"
#include "ptx.cuh"

namespace cfb {
namespace {

constexpr int kStreamWarps = 8;
constexpr int kStreamFeatures = 16;
constexpr int kStreamLeast = 8;  // features of a CTA, where there are so few
constexpr int kStreamThreads = (kStreamWarps + 1) * kWarp;
constexpr int kStreamBoxBytes = kStreamFeatures * 128;

constexpr int kStreamTokens = 8;
constexpr int kStreamTokenBoxBytes = kStreamTokens * 128;
constexpr int kStreamRedRow = kStreamFeatures + 1;
constexpr int kStreamRedFloats = kStreamWarps * kStreamTokens * kStreamRedRow;

// Shared memory: the stages' blocks of weights and tokens, their scales, the sums of a
// tile twice, barriers. Two CTAs on an SM, 113 KB each.
template <class Op>
struct StreamCfg {
  static constexpr int kTokenBytes = Op::kBlocks * kStreamTokenBoxBytes;
  static constexpr int kStageBytes = kStreamWarps * kStreamBoxBytes + kTokenBytes;
  static constexpr int kRedBytes = 2 * kStreamRedFloats * 4;
  static constexpr int kStages =
      (115712 - 1024 - 128 - kRedBytes) / (kStageBytes + Op::kScaleBytes);
  static constexpr int kScales = kStages * kStageBytes;
  static constexpr int kRed = kScales + kStages * Op::kScaleBytes;
  static constexpr int kBars = kRed + kRedBytes;
  static constexpr size_t kSmem = 1024 + kBars + 128;
  static_assert(Op::kBlocks * Op::kMatrices == kStreamWarps);
  static_assert(kSmem <= 115712 && kBars % 8 == 0 && kScales % 128 == 0);
};

// The fragments of a block: rows g and g + 8, the two 16-byte halves of 32 bytes.
struct StreamRows {
  uint4 w[2][2];
};

// The tiles of n features: as many to each CTA, and all of one size or one less. A
// tile takes a CTA the same time whatever its size (what is in flight is a number of
// stages), so a last round of full tiles for some of the CTAs would cost as much as
// one for all.
struct StreamTiles {
  int count, grid, rows;  // rows: the larger size
  int larger;             // the first tiles, of that size
  __device__ __forceinline__ int first(int tile) const {
    return tile * (rows - 1) + min(tile, larger);
  }
};

inline StreamTiles stream_tiles(int64_t n) {
  StreamTiles t;
  t.grid =
      static_cast<int>(std::min<int64_t>((n + kStreamLeast - 1) / kStreamLeast, 2 * sm_count()));
  const int64_t a_round = int64_t{t.grid} * kStreamFeatures;
  t.count = static_cast<int>((n + a_round - 1) / a_round * t.grid);
  t.rows = static_cast<int>((n + t.count - 1) / t.count);
  t.larger = static_cast<int>(n - int64_t{t.count} * (t.rows - 1));
  return t;
}

// The tensor maps of one operand, [rows, k] in blocks of 128 bytes. The first
// `whole_steps` stages come in one copy, [block][row]: the copies' number is what bounds
// these kernels otherwise (eight boxes of 16 x 128 bytes a stage: 115 cycles a box,
// however many of its rows exist). A last stage with part of a block, which such a map
// cannot describe, takes a copy for each block, `pitch` rows apart.
struct StreamMap {
  CUtensorMap tm, tm_block;

  int make(const void *base, int esize, int64_t k, int64_t n, int rows, int blocks,
           int whole_steps) {
    int st = CF_OK;
    if (whole_steps > 0) st = make_block_map(&tm, base, esize, k, n, rows, blocks);
    if (st == CF_OK && k * esize % 128 != 0) {
      st = make_map(&tm_block, base, esize, k, n, 128 / esize, rows, true);
    }
    return st;
  }

  // By a whole warp: block `block` and those after it, as the mask `exist` says.
  template <int kBlocks, int kPitch, int kBlockElems>
  __device__ __forceinline__ void load(uint8_t *dst, uint64_t *bar, int row, int block,
                                       unsigned exist, bool whole) const {
    const int lane = static_cast<int>(threadIdx.x) % kWarp;
    if (whole) {
      if (lane == 0) ptx::tma_load_3d(dst, &tm, bar, 0, row, block);
    } else if (lane < kBlocks && (exist >> lane & 1u)) {
      ptx::tma_load_2d(dst + lane * kPitch * 128, &tm_block, bar, (block + lane) * kBlockElems,
                       row);
    }
  }
};

// Stages that are copied whole: all of them where k is whole blocks (what is beyond k is
// zeros then).
inline int stream_whole_steps(int64_t k_bytes, int blocks) {
  return static_cast<int>(k_bytes % 128 == 0 ? (k_bytes / 128 + blocks - 1) / blocks
                                             : k_bytes / 128 / blocks);
}

// Op: what is multiplied. kMatrices of weights share the warps, kBlocks of 128 bytes of
// k (kBlockElems elements) a stage for each, of the same tokens. w[matrix] and
// less[matrix], the maps of a tile's rows and of one row less, tokens, token_rows,
// blocks (of k); tiles, steps (stages of a tile), whole_steps, err. kScaleBytes of the tokens'
// scales by load_scales(dst, bar, step), scale_bytes of them copied, or none.
// Weights, the weights' scales of a lane: fetch(weights, feature, step, warp) at every
// 32nd step for the next 32, ahead of the tile; multiply(rows, token words, scales,
// weights, feature, step, acc); store(feature, count, red) by all consumer threads, of
// a tile's first `count` features. What the rows beyond them hold reaches only sums
// that are not stored.
template <class Op>
__global__ void __launch_bounds__(kStreamThreads, 2)
    stream_kernel(const __grid_constant__ Op op) {
  using C = StreamCfg<Op>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::kBars);
  uint64_t *empty = full + C::kStages;
  int *abort_flag = reinterpret_cast<int *>(empty + C::kStages);
  const int warp = threadIdx.x / kWarp;
  const int lane = threadIdx.x % kWarp;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], kStreamWarps);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();

  if (warp == kStreamWarps) {
    uint32_t outstanding = 0, parities = 0;
    int tile = blockIdx.x, step = 0, stage = 0;
    uint32_t phase = 0;
    int feature, count;  // of the tile
    auto locate = [&] {
      feature = op.tiles.first(tile);
      count = op.tiles.first(tile + 1) - feature;
    };
    locate();
    auto exist = [&] {
      return (1u << min(Op::kBlocks, op.blocks - step * Op::kBlocks)) - 1u;
    };
    auto weights = [&] {
      // Whole stages are filled up with zeros.
      const int copied = step < op.whole_steps ? Op::kBlocks : __popc(exist());
      if (lane == 0) {
        ptx::mbar_expect_tx(&full[stage],
                            copied * (Op::kMatrices * count + op.token_rows) * 128 +
                                op.scale_bytes);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < Op::kMatrices; ++i) {
        (count < op.tiles.rows ? op.less[i] : op.w[i])
            .template load<Op::kBlocks, kStreamFeatures, Op::kBlockElems>(
                smem + stage * C::kStageBytes + i * Op::kBlocks * kStreamBoxBytes, &full[stage],
                feature, step * Op::kBlocks, exist(), step < op.whole_steps);
      }
      outstanding |= 1u << stage;
      parities = (parities & ~(1u << stage)) | (phase << stage);
    };
    auto tokens = [&] {
      op.tokens.template load<Op::kBlocks, kStreamTokens, Op::kBlockElems>(
          smem + stage * C::kStageBytes + kStreamWarps * kStreamBoxBytes, &full[stage], 0,
          step * Op::kBlocks, exist(), step < op.whole_steps);
      if constexpr (Op::kScaleBytes > 0) {
        if (lane == 0) {
          op.load_scales(smem + C::kScales + stage * Op::kScaleBytes, &full[stage], step);
        }
      }
    };
    auto advance = [&] {
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1;
      }
      if (++step == op.steps) {
        step = 0;
        tile += gridDim.x;
        locate();
      }
    };
    // The first round of weights is on its way before the tokens are there.
    for (int i = 0; i < C::kStages && tile < op.tiles.count; ++i, advance()) weights();
    ptx::grid_dep_wait();
    tile = blockIdx.x, step = 0, stage = 0, phase = 0;
    locate();
    for (int i = 0; i < C::kStages && tile < op.tiles.count; ++i, advance()) tokens();
    for (; tile < op.tiles.count && !aborted(abort_flag); advance()) {
      if (!ptx::mbar_wait(&empty[stage], phase ^ 1)) {
        record_timeout(op.err, abort_flag);
        break;
      }
      weights();
      tokens();
    }
    if (aborted(abort_flag)) {
      for (int s = 0; s < C::kStages; ++s) {
        if (outstanding & (1u << s)) ptx::mbar_wait(&full[s], (parities >> s) & 1u, 200000000ull);
      }
    }
    return;
  }

  const int g = lane / 4, t = lane % 4;
  const int block = warp % Op::kBlocks;  // of a stage's, in matrix warp / kBlocks
  const uint32_t base = ptx::smem_addr(smem);
  int feature = op.tiles.first(blockIdx.x);
  typename Op::Weights cur, next;
  op.fetch(next, feature, 0, warp);
  int stage = 0, parity = 0;
  uint32_t phase = 0;
  for (int tile = blockIdx.x; tile < op.tiles.count; tile += gridDim.x, parity ^= 1) {
    const int count = op.tiles.first(tile + 1) - feature;
    const int after = op.tiles.first(min(tile + static_cast<int>(gridDim.x), op.tiles.count));
    float acc[4] = {};
    for (int step = 0; step < op.steps; ++step) {
      if (step % kWarp == 0) {
        cur = next;
        if (step + kWarp < op.steps) {
          op.fetch(next, feature, step + kWarp, warp);
        } else {
          op.fetch(next, after, 0, warp);
        }
      }
      // After a wait that gave up the rest runs through on what is there, so
      // that no warp waits for another at the tile's end.
      if (!aborted(abort_flag) && !ptx::warp_wait(&full[stage], phase) && lane == 0) {
        record_timeout(op.err, abort_flag);
      }
      if (step * Op::kBlocks + block < op.blocks) {
        const uint32_t in_stage = base + stage * C::kStageBytes;
        const uint32_t tokens = in_stage + kStreamWarps * kStreamBoxBytes;
        const uint32_t weights = in_stage + (warp - block) * kStreamBoxBytes;
        const int row = block * (step < op.whole_steps ? count : kStreamFeatures) + g;
        const int token = block * (step < op.whole_steps ? op.token_rows : kStreamTokens) + g;
        StreamRows rows;
        uint4 x[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 16-byte chunks, swizzled by the row modulo 8
          const int chunk = 2 * t + h;
          rows.w[0][h] = ptx::ld_shared_v4(weights + row * 128 + ((chunk ^ (row & 7)) << 4));
          rows.w[1][h] = ptx::ld_shared_v4(weights + (row + 8) * 128 + ((chunk ^ (row & 7)) << 4));
          x[h] = ptx::ld_shared_v4(tokens + token * 128 + ((chunk ^ (token & 7)) << 4));
        }
        float s[2] = {1.0f, 1.0f};  // of the lane's two result columns, tokens 2t and 2t + 1
        if constexpr (Op::kScaleBytes > 0) {
          const uint32_t at = base + C::kScales + stage * Op::kScaleBytes +
                              (warp * kStreamTokens + 2 * t) * 4;
          s[0] = ptx::ld_shared_f32(at);
          s[1] = ptx::ld_shared_f32(at + 4);
        }
        ptx::warp_arrive(&empty[stage]);
        op.multiply(rows, x, s, cur, feature, step, acc);
      } else {
        ptx::warp_arrive(&empty[stage]);
      }
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // Two buffers, so one barrier a tile: a buffer is written again only after
    // the barrier of the tile in between.
    float *red = reinterpret_cast<float *>(smem + C::kRed) + parity * kStreamRedFloats;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      red[(warp * kStreamTokens + 2 * t + (i & 1)) * kStreamRedRow + g + (i & 2) * 4] = acc[i];
    }
    ptx::named_bar_sync(1, kStreamWarps * kWarp);
    op.store(feature, count, red);
    feature = after;
  }
}

// `dependent`: may start while the kernel launched just before it still runs
// (it waits for that one before it reads tokens).
template <class Op>
int launch_stream(const Op &op, bool dependent, cudaStream_t s) {
  if (int st = allow_dynamic_smem<stream_kernel<Op>>(StreamCfg<Op>::kSmem)) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(op.tiles.grid));
  cfg.blockDim = dim3(kStreamThreads);
  cfg.dynamicSmemBytes = StreamCfg<Op>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  set_programmatic_dependency(attr[0]);
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  CFB_TRY_CUDA(cudaLaunchKernelEx(&cfg, stream_kernel<Op>, op));
  return check_launch();
}

}  // namespace
}  // namespace cfb
