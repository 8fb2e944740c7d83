// Runs csrc/row_ring.cuh on the host over a model of mbarriers and bulk copies: the row
// loop of a persistent CTA's first thread, with a wait that gives up at each row in turn.
// Afterwards no copy may be in flight, whatever row it was.
//
// The model: a barrier counts its completed phases; a copy, once issued, is in flight
// until someone waits for the phase that it completes, or until the next round of waits
// finds it landed. A wait for a parity that the barrier has passed returns at once.
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#define __device__
#define __forceinline__ inline

static int g_fail_at = -1;  // this wait of the row loop gives up
static int g_waits = 0;
static bool g_draining = false;

struct Barrier {
  int phase = 0;
  bool in_flight = false;
};
static Barrier g_bars[8];
static uint64_t g_full[8];

static Barrier &model(const uint64_t *bar) { return g_bars[bar - g_full]; }

static unsigned atomicOr(unsigned *p, unsigned v) {
  const unsigned old = *p;
  *p |= v;
  return old;
}

namespace cfb {
enum DeviceError : unsigned { kDevErrTimeout = 1u };
namespace ptx {
static void mbar_init(uint64_t *bar, uint32_t) { model(bar) = Barrier{}; }
static void fence_mbar_init() {}
static void mbar_expect_tx(uint64_t *bar, uint32_t) {
  if (model(bar).in_flight) {
    std::puts("a stage is filled while its copy is in flight");
    std::exit(1);
  }
  model(bar).in_flight = true;
}
static void bulk_load(void *, const void *, uint32_t, uint64_t *) {}
static bool mbar_wait(uint64_t *bar, uint32_t parity, uint64_t = 0) {
  Barrier &b = model(bar);
  if ((b.phase & 1) != static_cast<int>(parity)) return true;  // that phase has passed
  if (!g_draining && g_waits++ == g_fail_at) return false;
  if (!b.in_flight) {
    std::puts("a wait for a copy that nobody issued");
    std::exit(1);
  }
  b.in_flight = false;
  ++b.phase;
  return true;
}
}  // namespace ptx
}  // namespace cfb

#include "row_ring.cuh"

int main() {
  int runs = 0, left = 0;
  for (int stages = 1; stages <= 4; ++stages) {
    for (int rows = 1; rows <= 13; ++rows) {
      for (int fail = -1; fail < rows; ++fail) {
        unsigned err = 0;
        g_fail_at = fail;
        g_waits = 0;
        g_draining = false;
        uint8_t src[4] = {}, smem[64];
        cfb::RowRing<1> ring;
        ring.src[0] = src;
        ring.smem = smem;
        ring.full = g_full;
        ring.err = &err;
        ring.row_bytes = 0;
        ring.stages = stages;
        ring.init();
        for (int s = 0; s < stages && s < rows; ++s) ring.issue(s, s);
        for (int row = 0; row < rows; ++row) {
          ring.wait();
          if (row + stages < rows) ring.issue(ring.stage, row + stages);
          ring.advance();
        }
        g_draining = true;
        ring.drain();
        ++runs;
        if ((err != 0) != (fail >= 0)) {
          std::printf("%d stages, %d rows, failure at %d: error word %u\n", stages, rows, fail, err);
          return 1;
        }
        for (int s = 0; s < stages; ++s) {
          if (g_bars[s].in_flight) {
            ++left;
            std::printf("%d stages, %d rows, failure at row %d: stage %d still in flight\n", stages,
                        rows, fail, s);
          }
        }
      }
    }
  }
  std::printf("%d runs, %d copies left in flight\n", runs, left);
  return left != 0;
}
