// A ring of rows in shared memory, filled by bulk copies.
#pragma once

#include "cf_common.cuh"
#include "ptx.cuh"

namespace cfb {
namespace {

// The ring of one group of threads: each stage holds a row of up to
// kArrays inputs. Thread 0 of the group issues the copies; every thread waits.
// A wait that runs out records the error and stops all later waits and copies
// of the thread, and the kernel runs to its end on what is there.
template <int kArrays>
struct RowRing {
  const uint8_t *src[kArrays];  // null: not read
  uint8_t *smem;
  uint64_t *full;
  unsigned *err;
  uint32_t row_bytes;
  int stages, stage = 0;
  uint32_t phase = 0, outstanding = 0;
  bool failed = false;

  __device__ __forceinline__ void init() {
    for (int s = 0; s < stages; ++s) ptx::mbar_init(&full[s], 1);
    ptx::fence_mbar_init();
  }

  __device__ __forceinline__ void issue(int to, int64_t row) {
    if (failed) return;
    uint32_t bytes = 0;
#pragma unroll
    for (int i = 0; i < kArrays; ++i) bytes += src[i] ? row_bytes : 0;
    ptx::mbar_expect_tx(&full[to], bytes);
#pragma unroll
    for (int i = 0; i < kArrays; ++i) {
      if (src[i]) {
        ptx::bulk_load(smem + (to * kArrays + i) * row_bytes, src[i] + row * row_bytes, row_bytes,
                       &full[to]);
      }
    }
    outstanding |= 1u << to;
  }

  // Waits for the current stage.
  __device__ __forceinline__ void wait() {
    if (!failed && !ptx::mbar_wait(&full[stage], phase)) {
      atomicOr(err, kDevErrTimeout);
      failed = true;
    }
    if (!failed) outstanding &= ~(1u << stage);
  }

  template <typename T>
  __device__ __forceinline__ const T *row(int array) const {
    return reinterpret_cast<const T *>(smem + (stage * kArrays + array) * row_bytes);
  }

  // A thread whose wait gave up stays where it was: drain() reads from there which
  // phase each outstanding copy completes.
  __device__ __forceinline__ void advance() {
    if (failed) return;
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }

  // After a failed wait: lets copies in flight land before the CTA's shared
  // memory goes away (bounded).
  __device__ __forceinline__ void drain() {
    if (!failed) return;
    for (int s = 0; s < stages; ++s) {
      if (outstanding & (1u << s)) {
        ptx::mbar_wait(&full[s], s < stage ? phase ^ 1 : phase, 200000000ull);
      }
    }
  }
};

}  // namespace
}  // namespace cfb
