"""The turns that two query tiles take on the exponential unit, from item to item: the rules are
read out of the attention kernels' sources, those of a warp whose bounded wait ran out among them,
and walked on the host in every order that chance brings. A named barrier of 64 threads is complete with any two warps' arrivals, so a warp
that arrives twice before its partner has waited leaves the partner, whose wait has no limit,
without an arrival."""
import random
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "svod_b200" / "csrc"
KERNELS = ["attention_tc_p.cu", "attention_paged_tc.cu", "attention_tc.cu"]
ONE_ITEM = "attention_tc.cu"  # an item a CTA: its last turn is nobody's to wait for


def rules(name, call):
    """The conditions under which the kernel makes `call`, as Python."""
    lines = [line for line in (CSRC / name).read_text().splitlines() if not line.strip().startswith("//")]
    found = []
    for k, line in enumerate(lines):
        if call not in line:
            continue
        conds = re.findall(r"if \((.*)\)", line.split("named_barrier")[0])
        if re.search(r"if \(.*[{)]$", lines[k - 1]):  # the block it stands in, or the line it goes with
            conds.append(re.search(r"if \((.*)\)", lines[k - 1]).group(1))
        found.append(" and ".join(f"({c})" for c in conds).replace("||", " or ").replace("&&", " and ") or "True")
    return found


@pytest.mark.parametrize("name", KERNELS)
@pytest.mark.parametrize("seed", range(60))
def test_no_warp_arrives_twice_before_its_partner_waits(name, seed):
    g = random.Random(seed)
    items = [g.choice([0, 1, 1, 2, 3, 7]) for _ in range(1 if name == ONE_ITEM else g.randint(2, 25))]
    waits, passes = rules(name, "named_barrier(my_turn"), rules(name, "named_barrier_arrive(other_turn")
    border = {w for w in waits if "turned" in w}  # once an item
    waits = [w for w in waits if w not in border]  # once a turn: in the block loop, and where a warp has given up
    assert waits and len(border) <= 1
    assert len(waits) == len(passes), "a place that passes turns on without waiting for its own"

    def walk(i):
        turns = 0
        for n_paired in items:
            env = dict(i=i, n_paired=n_paired, pairs=n_paired, turned=turns > 0)
            if any(eval(b, {}, env) for b in border):
                yield "wait"
            for n in range(n_paired):
                env.update(n=n, m=n, turns=turns)
                must, may = {eval(w, {}, env) for w in waits}, {eval(p, {}, env) for p in passes}
                assert len(must) == len(may) == 1, "a warp that gave up walks other turns"
                if must.pop():
                    yield "wait"
                if may.pop():
                    yield "pass"
                turns += 1

    steps, at, arrived = [list(walk(0)), list(walk(1))], [0, 0], [0, 0]
    while at[0] < len(steps[0]) or at[1] < len(steps[1]):
        able = [i for i in (0, 1) if at[i] < len(steps[i]) and (steps[i][at[i]] == "pass" or arrived[i] > 0)]
        assert able, "both wait"
        i = g.choice(able)
        if steps[i][at[i]] == "wait":
            arrived[i] -= 1
        else:
            arrived[1 - i] += 1
            assert arrived[1 - i] <= 1, "two arrivals before the partner has waited"
        at[i] += 1
