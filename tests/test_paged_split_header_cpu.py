"""The arithmetic by which the CTAs of the paged attention share their work out, as the kernel
compiles it (csrc/paged_split.cuh), built for the host and compared with a walk of its own."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

from tests.test_paged_split_cpu import BLOCK, COST, LEAST, Plan

CSRC = Path(__file__).resolve().parent.parent / "svod_b200" / "csrc"

HOST = """
#include "paged_split.cuh"
using namespace svodb::paged;
struct Seen { int causal, has_window; int64_t win_left, win_right; };
struct Params { Seen a; int tile_tokens; };
extern "C" int constants(int* out) { out[0] = kItemCost, out[1] = kLeastShare, out[2] = kBlockKeys; return 0; }
// The shares of a CTA, seven numbers each. The steps from item to item are the kernel's; the row in
// which the run begins is found one row after the other, where its warp adds up 32 at a time.
extern "C" int walk(int rows, const int* start, const int* n, int kv, int tile_tokens, int causal, int window, int left, int right,
                    int ctas, int cta, int* out, int room) {
  const Params p{{causal, window, left, right}, tile_tokens};
  auto row_at = [&](int b) { return Row{start[b], n[b], false}; };
  int64_t total = 0;
  for (int b = 0; b < rows; ++b) total += row_weight(p, row_at(b)) * kv;
  const Run run = run_of(total, cta, ctas);
  int count = 0, b = 0, hk, q;
  if (run.c0 >= run.c1) return 0;
  int64_t x = 0;
  while (x + row_weight(p, row_at(b)) * kv <= run.c0) x += row_weight(p, row_at(b++)) * kv;
  Row row = row_at(b);
  find_item(p, run, row, row_weight(p, row), x, hk, q);
  while (x < run.c1) {
    const int blocks = item_blocks(p, row, q), weight = blocks + kItemCost;
    const int from = share_from(run.c0, x), to = share_to(run.c1, x, weight);
    if (to > from) {
      if (count == room) return -1;
      const int all[7] = {b, hk, q, from, to, part_of(from, to, blocks), last_cta(x, weight, run.quota)};
      for (int i = 0; i < 7; ++i) out[count * 7 + i] = all[i];
      ++count;
    }
    x += weight;
    if (++q < live_items(p, row)) continue;
    q = 0;
    if (++hk < kv) continue;
    hk = 0;
    do {
      if (++b >= rows) return count;
      row = row_at(b);
    } while (row.n == 0);
  }
  return count;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    at = tmp_path_factory.mktemp("split")
    (at / "host.cpp").write_text(HOST)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow,bounds", "-fsanitize-undefined-trap-on-error", "-shared",
                    "-fPIC", f"-I{CSRC}", str(at / "host.cpp"), "-o", str(at / "host.so")], check=True)
    return C.CDLL(str(at / "host.so"))


def test_the_walk_has_the_kernels_constants(host):
    got = (C.c_int * 3)()
    host.constants(got)
    assert list(got) == [COST, LEAST, BLOCK]


@pytest.mark.parametrize("seed", range(200))
def test_the_kernels_shares_are_the_walks(host, seed):
    """The cases of the Python walk, whose own test shows that every block is taken once and that
    an item's parts lie where the merge looks; rows without tokens at either end among them."""
    g = random.Random(seed)
    rows = [(g.choice([0, g.randint(0, 5000)]), g.choice([0, 1, g.randint(1, 900)])) for _ in range(g.randint(1, 9))]
    kv, step, causal = g.choice([1, 2, 5, 8]), g.choice([256, 128, 84, 32, 2]), g.random() < 0.7
    window, ctas = g.choice([None, None, (0, 0), (40, 0), (700, 64)]), g.choice([148, 148, 3, 1])
    if seed % 3 == 0:
        rows = [(7, 0)] + rows + [(0, 0), (90, 0)]
    plan = Plan(rows, kv, step, causal, window, ctas)
    ints = lambda xs: (C.c_int * len(xs))(*xs)
    starts, ns, out = ints([r[0] for r in rows]), ints([r[1] for r in rows]), (C.c_int * (7 * 40000))()
    for cta in range(ctas):
        n = host.walk(len(rows), starts, ns, kv, step // 2, causal, window is not None, *(window or (0, 0)), ctas, cta, out, 40000)
        got = [tuple(out[7 * k:7 * k + 7]) for k in range(n)]
        want, split = plan.walk(cta)
        assert [s[:6] for s in got] == want
        first = [(*s[:3], s[6]) for s in got if s[5] == 1]
        assert first == ([split] if split else [])
