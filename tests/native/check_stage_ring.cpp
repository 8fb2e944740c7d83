// Runs csrc/stage_ring.cuh on the host over a model of its barriers: a producer fills any
// number of stages, the consumer's arrivals on `empty` stay under way until somebody
// waits for them. A producer that leaves on the usual way has to leave none under way, and
// one whose wait gave up no copies.
//
// `drop_wait`: the plain end of a producer that does not wait, to show that the model sees it.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#define __device__
#define __forceinline__ inline

// Phases completed, and whether what completes the next one is under way.
struct Barrier {
  int phase = 0;
  bool under_way = false;
};

constexpr int kMost = 8;
static uint64_t g_full[kMost], g_empty[kMost];
static Barrier g_landed[kMost], g_freed[kMost];
static int g_fail_at, g_waits;
static bool g_draining;

static void fail(const char *what) {
  std::puts(what);
  std::exit(1);
}

namespace cfb {
namespace ptx {
static bool mbar_wait(uint64_t *bar, uint32_t parity, uint64_t = 0) {
  const bool full = bar >= g_full && bar < g_full + kMost;
  const int s = static_cast<int>(bar - (full ? g_full : g_empty));
  Barrier &b = full ? g_landed[s] : g_freed[s];
  if ((b.phase & 1) != static_cast<int>(parity)) return true;  // that phase has passed
  if (!full && !g_draining && g_waits++ == g_fail_at) return false;
  if (!b.under_way) fail("a wait for what nobody issued");
  if (!full) {
    // The MMAs retired, which their operands' copies preceded.
    g_landed[s].under_way = false;
    ++g_landed[s].phase;
  }
  b.under_way = false;
  ++b.phase;
  return true;
}
}  // namespace ptx
}  // namespace cfb

#include "stage_ring.cuh"

static int g_left = 0;

template <int kStages>
static void run(int fills, int fail_at, bool drop_wait) {
  for (int s = 0; s < kMost; ++s) g_landed[s] = g_freed[s] = Barrier{};
  g_fail_at = fail_at;
  g_waits = 0;
  g_draining = false;
  cfb::StageRing<kStages> ring;
  bool ok = true;
  for (int i = 0; i < fills && ok; ++i) {
    ok = ring.wait_free(g_empty);
    if (!ok) break;
    if (ring.stage != i % kStages) fail("stages out of order");
    if (g_landed[ring.stage].under_way || g_freed[ring.stage].under_way) fail("a stage in use");
    g_landed[ring.stage].under_way = true;
    g_freed[ring.stage].under_way = true;
    ring.filled();
  }
  if (ok && !drop_wait) ok = ring.wait_all_free(g_empty);
  if (!ok) {
    g_draining = true;
    ring.drain(g_full);
  }
  for (int s = 0; s < kStages; ++s) {
    if (g_landed[s].under_way && !drop_wait) {
      ++g_left;
      std::printf("%d stages, %d fills, failure at %d: copies of stage %d under way\n", kStages,
                  fills, fail_at, s);
    }
    if (ok && g_freed[s].under_way) ++g_left;
  }
}

template <int kStages>
static void all(bool drop_wait) {
  for (int fills = 0; fills <= 3 * kStages + 2; ++fills) {
    run<kStages>(fills, -1, drop_wait);
    for (int at = 0; at < fills && !drop_wait; ++at) run<kStages>(fills, at, false);
  }
}

int main(int argc, char **argv) {
  const bool drop_wait = argc > 1 && std::strcmp(argv[1], "drop_wait") == 0;
  all<1>(drop_wait);
  all<2>(drop_wait);
  all<4>(drop_wait);
  all<6>(drop_wait);
  std::printf("%d left under way\n", g_left);
  return g_left != 0;
}
