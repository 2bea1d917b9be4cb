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
// The shares of a CTA, eight numbers each; the row in which its run begins is found one row after
// the other, where the kernel's warp adds up 32 at a time.
extern "C" int walk(int rows, const int* start, const int* n, int kv, int tile_tokens, int causal, int window, int left, int right,
                    int ctas, int cta, int* out, int room) {
  const Params p{{causal, window, left, right}, tile_tokens};
  auto row_at = [&](int b) { return Row{start[b], n[b], false}; };
  int64_t total = 0;
  for (int b = 0; b < rows; ++b) total += row_weight(p, row_at(b)) * kv;
  const Run run = run_of(total, cta, ctas);
  int count = 0;
  if (run.c0 >= run.c1) return 0;
  int64_t x = 0;
  int b = 0;
  while (x + row_weight(p, row_at(b)) * kv <= run.c0) x += row_weight(p, row_at(b++)) * kv;
  walk_run(p, run, rows, kv, b, x, row_weight(p, row_at(b)), row_at, [&](const Row& row, const Share& s) {
    int lo, hi;
    item_keys(p, row, s.q, lo, hi);
    const int all[8] = {s.b, s.hk, s.q, s.from, s.to, s.part, s.last_cta, s.blocks == (hi + kBlockKeys - 1) / kBlockKeys - lo / kBlockKeys};
    for (int i = 0; i < 8; ++i) out[count * 8 + i] = all[i];
    return ++count < room;
  });
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
    starts, ns, out = ints([r[0] for r in rows]), ints([r[1] for r in rows]), (C.c_int * (8 * 40000))()
    for cta in range(ctas):
        n = host.walk(len(rows), starts, ns, kv, step // 2, causal, window is not None, *(window or (0, 0)), ctas, cta, out, 40000)
        got = [tuple(out[8 * k:8 * k + 8]) for k in range(n)]
        want, split = plan.walk(cta)
        assert [s[:6] for s in got] == want and all(s[7] == 1 for s in got)
        first = [(*s[:3], s[6]) for s in got if s[5] == 1]
        assert first == ([split] if split else [])
