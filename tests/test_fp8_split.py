"""The exchange of partial sums between the CTAs that split a tile of the 8-bit product (csrc/fp8_split.h),
run on the host: every byte that a CTA is sent is one that it expects and waits for before it leaves."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashbfp_b200", "csrc")

# One tile: what each CTA (split, pair rank) expects, what the others send it, and whether a warp of it
# waits. features: whether blocks without features are left out (0: the control, in which they are
# sent and counted although nobody adds them).
HARNESS = r"""
#include "fp8_split.h"
#include <string.h>
using namespace fbfp;
static bool live(int features, int64_t t, int64_t f, int64_t m, int64_t n) {
  return features ? block_live(t, f, m, n) : t < m;
}
extern "C" int tile(int cg, int splits, int64_t tok, int64_t f0, int64_t m, int64_t n, int features) {
  int bad = 0;
  for (int pr = 0; pr < cg; ++pr) {
    const int64_t t0 = tok + 128 * pr;
    for (int owner = 0; owner < splits; ++owner) {
      int want = features ? owned_blocks(owner, splits, t0, f0, m, n) : 0, got = 0;
      bool waits = false, used[14];
      memset(used, 0, sizeof used);
      for (int q = 0; q < 4; ++q)
        for (int c = 0; c < 4; ++c) {
          if (block_owner(q, c, splits) != owner) continue;
          const int64_t t = t0 + 32 * q, f = f0 + 32 * c;
          if (!features && t < m) ++want;
          waits |= block_live(t, f, m, n);
          for (int sp = 0; sp < splits; ++sp) {
            if (sp == owner || !live(features, t, f, m, n)) continue;
            const int room = block_slot(q, c, splits) * (splits - 1) + (sp < owner ? sp : sp - 1);
            if (room >= 14 || used[room]) bad |= 1;          // a room of its own
            else used[room] = true;
            ++got;
          }
        }
      if (got != want * (splits - 1)) bad |= 2;             // what is sent is what is expected
      if (got && !waits) bad |= 4;                          // and somebody waits for it
    }
  }
  return bad;
}
// The accumulators' ring: the MMAs take halves in turn and wait, from the second use of a slot on,
// for its last drain; the epilogue drains in turn. all: every drain arrives (the control). Returns
// the arrivals that nobody waited for, or -1 if a wait would never end.
extern "C" int64_t ring(int64_t halves, int ring, int all) {
  int64_t arrived[8] = {0}, waited[8] = {0};
  for (int64_t h = 0; h < halves; ++h) {
    const int slot = (int)(h % ring);
    if (h >= ring && arrived[slot] < ++waited[slot]) return -1;
    arrived[slot] += all || arrival_awaited(h, ring, halves);
  }
  int64_t rest = 0;
  for (int i = 0; i < ring; ++i) rest += arrived[i] - waited[i];
  return rest;
}
// A pair's stages after a failure: each stage's barrier counts one arrival and the bytes of both CTAs.
// `mine` and `other` loads were issued; fix: whether the first CTA makes up the difference. Returns how
// many of the last `stages` loads' phases never complete, whatever the order of the copies.
extern "C" int pair_loads(int64_t mine, int64_t other, int stages, int fix) {
  const int64_t most = mine > other ? mine : other;
  int open = 0;
  for (int64_t j = most > stages ? most - stages : 0; j < most; ++j) {
    const int64_t bytes = 1000 + j % 5;                     // of one CTA; they differ from load to load
    int64_t pending = 1, tx = 0;
    if (j < mine) { --pending; tx += 2 * bytes; tx -= bytes; }
    if (j < other) tx -= bytes;
    if (fix && loads_owed(j, mine, other) > 0) { --pending; tx += bytes; }
    if (fix && loads_owed(j, mine, other) < 0) tx -= bytes;
    open += pending != 0 || tx != 0;
  }
  return open;
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("split")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(d / "h.cpp"), "-o",
                    str(d / "h.so")], check=True)
    lib = ctypes.CDLL(str(d / "h.so"))
    lib.tile.argtypes = [ctypes.c_int, ctypes.c_int] + [ctypes.c_int64] * 4 + [ctypes.c_int]
    lib.pair_loads.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    lib.ring.argtypes, lib.ring.restype = [ctypes.c_int64, ctypes.c_int, ctypes.c_int], ctypes.c_int64
    return lib


@pytest.fixture(scope="module")
def tile(rules):
    return rules.tile


@pytest.mark.parametrize("halves_per_tile", [1, 2])
def test_no_arrival_is_left_over(rules, halves_per_tile):
    """Drained accumulators are reported to a pair's first CTA exactly as often as its MMAs wait."""
    ring = halves_per_tile + 1
    for tiles in list(range(1, 40)) + [1000]:
        assert rules.ring(tiles * halves_per_tile, ring, 0) == 0
        assert rules.ring(tiles * halves_per_tile, ring, 1) == min(ring, tiles * halves_per_tile)     # the control


def tiles(m, n, cg):
    return [(t, f) for t in range(0, m, 128 * cg) for f in range(0, n, 128)]


@pytest.mark.parametrize("cg,splits", [(1, 2), (1, 4), (1, 8), (2, 2), (2, 4)])
def test_what_is_sent_is_waited_for(tile, cg, splits):
    for m in (65, 96, 97, 100, 128, 129, 200, 256, 257, 333):
        for n in (1, 31, 32, 33, 64, 65, 96, 97, 127, 128, 129, 200, 300, 1999, 2000, 4160):
            for t, f in tiles(m, n, cg):
                assert tile(cg, splits, t, f, m, n, 1) == 0, (m, n, t, f)


def test_blocks_without_features_would_be_sent_to_nobody(tile):
    """The control: counted by tokens alone, CTAs are sent sums that none of their warps waits for."""
    for m, n, cg, splits in ((90, 200, 1, 8), (100, 2000, 1, 4), (128, 4160, 1, 4), (333, 1999, 2, 4)):
        assert any(tile(cg, splits, t, f, m, n, 0) & 4 for t, f in tiles(m, n, cg)), (m, n)
        assert all(tile(cg, splits, t, f, m, n, 1) == 0 for t, f in tiles(m, n, cg))


@pytest.mark.parametrize("stages", [4, 6, 8])
def test_copies_of_a_pair_that_gave_up_all_land(rules, stages):
    """Whichever CTA of a pair got further (by at most the ring), every load's phase completes."""
    for mine in range(0, 30):
        for other in range(max(0, mine - stages), mine + stages + 1):
            assert rules.pair_loads(mine, other, stages, 1) == 0, (mine, other)
            assert (rules.pair_loads(mine, other, stages, 0) > 0) == (mine != other)       # the control
