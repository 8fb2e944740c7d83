// The producer's side of a ring of operand stages: which stage is filled next, what is
// in flight, and how the ring is left.
#pragma once

#include "ptx.cuh"

namespace cfb {
namespace {

// full[s] completes when a stage's copies have landed, empty[s] when the MMAs that read
// them have retired. One thread holds this.
template <int kStages>
struct StageRing {
  int stage = 0;
  uint32_t phase = 0, outstanding = 0, parities = 0;

  // Waits until the current stage may be filled; false if the wait gave up.
  __device__ __forceinline__ bool wait_free(uint64_t *empty) const {
    return ptx::mbar_wait(&empty[stage], phase ^ 1);
  }

  // The current stage's copies have been issued.
  __device__ __forceinline__ void filled() {
    outstanding |= 1u << stage;
    parities = (parities & ~(1u << stage)) | (phase << stage);
    advance();
  }

  // After the last stage: waits until all that were filled are free again. The MMAs'
  // arrivals on `empty` are asynchronous and reach both CTAs of a pair; one that nobody
  // has waited for could land in shared memory that its CTA no longer owns.
  __device__ __forceinline__ bool wait_all_free(uint64_t *empty) {
#pragma unroll 1
    for (int s = 0; s < kStages; ++s) {
      if (!wait_free(empty)) return false;
      advance();
    }
    return true;
  }

  // After a wait that gave up: lets copies in flight land (bounded).
  __device__ __forceinline__ void drain(uint64_t *full) const {
    for (int s = 0; s < kStages; ++s) {
      if (outstanding & (1u << s)) ptx::mbar_wait(&full[s], (parities >> s) & 1u, 200000000ull);
    }
  }

  __device__ __forceinline__ void advance() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

}  // namespace
}  // namespace cfb
