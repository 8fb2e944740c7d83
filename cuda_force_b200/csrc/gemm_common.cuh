// Pieces shared by the tensor-core kernels: operand descriptors, the abort
// protocol of their bounded waits, tile order, tensor maps and launch attributes.
#pragma once

#include <cuda.h>

#include <atomic>

#include "cf_common.cuh"
#include "ptx.cuh"

namespace cfb {
namespace {

__device__ __forceinline__ uint32_t swizzle_for_row_bytes(int row_bytes) {
  return row_bytes >= 128 ? ptx::kSwizzle128B : row_bytes == 64 ? ptx::kSwizzle64B
                                                                 : ptx::kSwizzle32B;
}

// Shared-memory descriptor of a K-major operand whose rows are `row_bytes`
// (32/64/128) long and swizzled at that width; 8-row core groups are
// 8 * row_bytes apart. k-step `ks` (16 elements = 32 bytes) advances the start
// address inside the swizzle atom.
__device__ __forceinline__ uint64_t kmajor_desc(uint32_t base, int row_bytes, int ks) {
  return ptx::make_smem_desc(base + ks * 32, 16, 8 * row_bytes, swizzle_for_row_bytes(row_bytes));
}

// Descriptor of an MN-major operand stored as chunks of `chunk_elems` MN
// elements (chunk_elems * 2 = row bytes, swizzled at that width) x k rows;
// chunks are `chunk_stride` bytes apart. k-step `ks` = 16 rows further.
__device__ __forceinline__ uint64_t mnmajor_desc(uint32_t base, int row_bytes, int chunk_stride,
                                                 int ks) {
  return ptx::make_smem_desc(base + ks * 16 * row_bytes, chunk_stride, 8 * row_bytes,
                             swizzle_for_row_bytes(row_bytes));
}

__device__ __forceinline__ void record_timeout(unsigned *err, int *abort_flag) {
  atomicOr(err, kDevErrTimeout);
  *reinterpret_cast<volatile int *>(abort_flag) = 1;
}

__device__ __forceinline__ bool aborted(const int *abort_flag) {
  return *reinterpret_cast<const volatile int *>(abort_flag) != 0;
}

// Tile t of a grid of `rows` x `cols` tiles, walked in bands of `band` rows
// with the row index fastest inside a band: the CTAs of one wave then share
// a few column blocks (each read from DRAM about once per band) while the
// band's row blocks stay resident in L2.
__device__ __forceinline__ void band_order(int t, int rows, int cols, int band, int &row,
                                           int &col) {
  const int per_band = band * cols;
  const int b = t / per_band;
  const int in_band = min(band, rows - b * band);
  const int i = t - b * per_band;
  row = b * band + i % in_band;
  col = i / in_band;
}

// The end of a product whose contracted dimension a cluster of `splits` CTAs has
// shared: each left its sums of the 128-row x kCols tile in fp32 at `part`, column
// by column. Every CTA adds its part of the columns over the shares, in rank
// order, and stores it as 16-bit numbers into y, the tile's first row, of which
// `rows` rows and columns [col0, cols) exist. A thread is a row, so its reads are
// its neighbours'. All threads of the cluster call this.
constexpr int kMaxSplits = 8;  // a portable cluster

template <int kCols, int kThreads, bool kBf16>
__device__ __forceinline__ void add_shares(uint32_t part, int share, int splits, uint16_t *y,
                                           int64_t ldy, int64_t rows, int64_t col0, int64_t cols) {
  constexpr int kRows = 128;
  constexpr int kGroups = kThreads / kRows;
  ptx::cluster_sync();
  const int row = static_cast<int>(threadIdx.x) % kRows;
  const int each = kCols / (splits * kGroups);  // columns of a thread
  const int first = (share * kGroups + static_cast<int>(threadIdx.x) / kRows) * each;
  if (threadIdx.x < kThreads && row < rows) {
    y += row * ldy;
    for (int c = first; c < first + each; c += 4) {  // all loads of four columns in flight
      float v[kMaxSplits][4];
#pragma unroll
      for (int r = 0; r < kMaxSplits; ++r) {
        const uint32_t from = ptx::map_shared_rank(part + (c * kRows + row) * 4,
                                                   static_cast<uint32_t>(r < splits ? r : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[r][j] = 0.0f;
          if (r < splits) v[r][j] = ptx::ld_shared_cluster_f32(from + j * kRows * 4);
        }
      }
#pragma unroll
      for (int r = 1; r < kMaxSplits; ++r) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[0][j] += v[r][j];
      }
      const uint32_t w[2] = {kBf16 ? ptx::pack_bf16x2(v[0][0], v[0][1])
                                   : ptx::pack_f16x2(v[0][0], v[0][1]),
                             kBf16 ? ptx::pack_bf16x2(v[0][2], v[0][3])
                                   : ptx::pack_f16x2(v[0][2], v[0][3])};
      const int64_t n = col0 + c;
      if (ldy % 4 == 0) {
        if (n < cols) *reinterpret_cast<uint2 *>(y + n) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (n + j < cols) y[n + j] = static_cast<uint16_t>(w[j / 2] >> (j % 2 * 16));
        }
      }
    }
  }
  ptx::cluster_sync();  // the others may still read this CTA's share
}

// CTAs that share each of `tiles` tiles: as many as the GPU has room for, with
// `least` blocks at least to each.
inline int split_count(int64_t tiles, int64_t blocks, int64_t least) {
  int splits = 1;
  while (splits < kMaxSplits && tiles * splits * 2 <= sm_count() && blocks >= splits * 2 * least) {
    splits *= 2;
  }
  return splits;
}

// ---- host: tensor maps and launches

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                   const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                   const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static std::atomic<EncodeTiledFn> cached{nullptr};
  EncodeTiledFn fn = cached.load(std::memory_order_acquire);
  if (fn != nullptr) return fn;
  void *sym = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) !=
          cudaSuccess ||
      q != cudaDriverEntryPointSuccess || sym == nullptr) {
    return nullptr;
  }
  fn = reinterpret_cast<EncodeTiledFn>(sym);
  cached.store(fn, std::memory_order_release);
  return fn;
}

// Launch attribute of the linear kernels: they may begin while the
// down-projection launched just before them on the stream is still running
// (their producers wait for it before reading P).
inline void set_programmatic_dependency(cudaLaunchAttribute &attr) {
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
}

inline CUtensorMapSwizzle swizzle_for(int inner_bytes) {
  switch (inner_bytes) {
    case 32: return CU_TENSOR_MAP_SWIZZLE_32B;
    case 64: return CU_TENSOR_MAP_SWIZZLE_64B;
    case 128: return CU_TENSOR_MAP_SWIZZLE_128B;
    default: return CU_TENSOR_MAP_SWIZZLE_NONE;
  }
}

inline int encode_map(CUtensorMap *map, const void *base, int esize, int rank,
                      const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                      bool swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return record_cuda_error(cudaErrorNotSupported);
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType dt = esize == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : esize == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                              : CU_TENSOR_MAP_DATA_TYPE_UINT32;
  const CUresult r =
      fn(map, dt, static_cast<cuuint32_t>(rank), const_cast<void *>(base), dims, strides, box, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE,
         swizzle ? swizzle_for(static_cast<int>(box[0]) * esize) : CU_TENSOR_MAP_SWIZZLE_NONE,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CF_OK : CF_ERR_UNSUPPORTED;
}

// 2-D row-major tensor [outer, inner] with element size esize and rows `ld` elements apart
// (0: inner), box [box_outer, box_inner].
inline int make_map(CUtensorMap *map, const void *base, int esize, int64_t inner, int64_t outer,
                    int box_inner, int box_outer, bool swizzle, int64_t ld = 0) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld ? ld : inner) * esize};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner),
                             static_cast<cuuint32_t>(box_outer)};
  return encode_map(map, base, esize, 2, dims, strides, box, swizzle);
}

// The same tensor, rows of whole 128-byte blocks, as [block][row][128 bytes]: a box of
// box_blocks blocks of box_rows rows, swizzled, in one copy.
inline int make_block_map(CUtensorMap *map, const void *base, int esize, int64_t inner,
                          int64_t outer, int box_rows, int box_blocks) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(128 / esize),
                              static_cast<cuuint64_t>(outer),
                              static_cast<cuuint64_t>(inner * esize / 128)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(inner) * esize, 128};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / esize),
                             static_cast<cuuint32_t>(box_rows),
                             static_cast<cuuint32_t>(box_blocks)};
  return encode_map(map, base, esize, 3, dims, strides, box, true);
}

}  // namespace
}  // namespace cfb
