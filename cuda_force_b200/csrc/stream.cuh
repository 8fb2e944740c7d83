// A product with up to eight tokens: bound by reading the weights once. Persistent CTAs
// walk over tiles of 16 output features; a producer warp streams the tiles' rows
// through a ring in shared memory by TMA, eight boxes of 16 rows x 128 bytes a
// stage, one for each of eight consumer warps. A consumer multiplies its box with
// all tokens on the warp-wide MMA (features as M, tokens as N): at these shapes
// the tensor core's rate does not matter. The warps' sums of a tile meet in
// shared memory. Two CTAs on an SM, so that one's tile ends hide behind the
// other's loads ([8, 8192] x [28672, 8192] in e4m3: 56 us, one CTA with twice the
// stages 66, the ring without any arithmetic 50).
//
// A lane's fragment words of a feature are 32 consecutive bytes of the box: any
// order of the contracted elements will do as long as both operands use it.
#pragma once

#include "cf_common.cuh"
#include "gemm_common.cuh"
#include "ptx.cuh"

namespace cfb {
namespace {

constexpr int kStreamWarps = 8;
constexpr int kStreamFeatures = 16;
constexpr int kStreamThreads = (kStreamWarps + 1) * kWarp;
constexpr int kStreamBoxBytes = kStreamFeatures * 128;
constexpr int kStreamStageBytes = kStreamWarps * kStreamBoxBytes;

constexpr int kStreamTokens = 8;
constexpr int kStreamStages = 6;
constexpr int kStreamRed = kStreamStages * kStreamStageBytes;
constexpr int kStreamRedRow = kStreamFeatures + 1;
constexpr int kStreamRedFloats = kStreamWarps * kStreamTokens * kStreamRedRow;
constexpr int kStreamBars = kStreamRed + 2 * kStreamRedFloats * 4;
constexpr size_t kStreamSmem = 1024 + kStreamBars + 128;
static_assert(kStreamSmem <= 115712, "two CTAs on an SM, 113 KB each");

// The fragments of a box: rows g and g + 8, the two 16-byte halves of 32 bytes.
struct StreamRows {
  uint4 w[2][2];
};

// Op: what is multiplied. tiles and steps (stages of a tile); boxes(step), how
// many of a stage's boxes exist; load_box(dst, bar, tile, step, box); Tokens with
// the tokens' operands of one box, fetched by load(tokens, tile, step, warp) a
// step ahead (it may be asked for a tile or box that does not exist);
// multiply(rows, tokens, acc); store(tile, red) by all consumer threads.
template <class Op>
__global__ void __launch_bounds__(kStreamThreads, 2)
    stream_kernel(const __grid_constant__ Op op) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kStreamBars);
  uint64_t *empty = full + kStreamStages;
  int *abort_flag = reinterpret_cast<int *>(empty + kStreamStages);
  const int warp = threadIdx.x / kWarp;
  const int lane = threadIdx.x % kWarp;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStreamStages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], kStreamWarps);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();

  if (warp == kStreamWarps) {
    // A lane for each box of a stage.
    int stage = 0;
    uint32_t phase = 0, outstanding = 0, parities = 0;
    for (int tile = blockIdx.x; tile < op.tiles && !aborted(abort_flag); tile += gridDim.x) {
      for (int step = 0; step < op.steps; ++step) {
        if (!ptx::mbar_wait(&empty[stage], phase ^ 1)) {
          record_timeout(op.err, abort_flag);
          break;
        }
        const unsigned boxes = op.boxes(step);  // a bit for each
        if (lane == 0) ptx::mbar_expect_tx(&full[stage], __popc(boxes) * kStreamBoxBytes);
        __syncwarp();
        if (lane < kStreamWarps && (boxes >> lane & 1u)) {
          op.load_box(smem + stage * kStreamStageBytes + lane * kStreamBoxBytes, &full[stage],
                      tile, step, lane);
        }
        outstanding |= 1u << stage;
        parities = (parities & ~(1u << stage)) | (phase << stage);
        if (++stage == kStreamStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (aborted(abort_flag)) {
      for (int s = 0; s < kStreamStages; ++s) {
        if (outstanding & (1u << s)) ptx::mbar_wait(&full[s], (parities >> s) & 1u, 200000000ull);
      }
    }
    return;
  }

  const int g = lane / 4, t = lane % 4;
  typename Op::Tokens next;
  op.begin();
  op.load(next, blockIdx.x, 0, warp);
  int stage = 0, parity = 0;
  uint32_t phase = 0;
  for (int tile = blockIdx.x; tile < op.tiles; tile += gridDim.x, parity ^= 1) {
    float acc[4] = {};
    for (int step = 0; step < op.steps; ++step) {
      const typename Op::Tokens cur = next;
      if (step + 1 < op.steps) {
        op.load(next, tile, step + 1, warp);
      } else {
        op.load(next, tile + static_cast<int>(gridDim.x), 0, warp);
      }
      // After a wait that gave up the rest runs through on what is there, so
      // that no warp waits for another at the tile's end.
      if (!aborted(abort_flag) && !ptx::warp_wait(&full[stage], phase) && lane == 0) {
        record_timeout(op.err, abort_flag);
      }
      if (op.boxes(step) >> warp & 1u) {
        const uint32_t row = ptx::smem_addr(smem + stage * kStreamStageBytes +
                                            warp * kStreamBoxBytes + g * 128);
        StreamRows rows;
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // the box is swizzled by its rows modulo 8
          const uint32_t chunk = static_cast<uint32_t>((2 * t + h) ^ g) << 4;
          rows.w[0][h] = ptx::ld_shared_v4(row + chunk);
          rows.w[1][h] = ptx::ld_shared_v4(row + 8 * 128 + chunk);
        }
        ptx::warp_arrive(&empty[stage]);
        op.multiply(rows, cur, acc);
      } else {
        ptx::warp_arrive(&empty[stage]);
      }
      if (++stage == kStreamStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // Two buffers, so one barrier a tile: a buffer is written again only after
    // the barrier of the tile in between.
    float *red = reinterpret_cast<float *>(smem + kStreamRed) + parity * kStreamRedFloats;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      red[(warp * kStreamTokens + 2 * t + (i & 1)) * kStreamRedRow + g + (i & 2) * 4] = acc[i];
    }
    ptx::named_bar_sync(1, kStreamWarps * kWarp);
    op.store(tile, red);
  }
}

// `dependent`: may start while the kernel launched just before it still runs
// (Op::begin waits for that one).
template <class Op>
int launch_stream(const Op &op, bool dependent, cudaStream_t s) {
  if (int st = allow_dynamic_smem<stream_kernel<Op>>(kStreamSmem)) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min(op.tiles, 2 * sm_count())));
  cfg.blockDim = dim3(kStreamThreads);
  cfg.dynamicSmemBytes = kStreamSmem;
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
