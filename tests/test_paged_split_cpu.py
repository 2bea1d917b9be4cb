"""How the CTAs of the paged attention share the work out (csrc/attention_paged_tc.cu), walked
on the host as the kernel walks it: every block of every item is taken once, an item's parts
lie where the merge looks for them, and no walk fails to end."""
import random

import pytest

COST, LEAST, BLOCK = 2, 4, 64  # kItemCost, kLeastShare and the keys of a block


def first_key(pos, window):
    return max(0, pos - window[0]) if window else 0


def last_key(pos, end, causal, window):
    x = end
    if causal:
        x = min(x, pos + 1)
    if window:
        x = min(x, pos + window[1] + 1)
    return x


class Plan:
    def __init__(self, rows, kv_heads, step, causal, window, ctas):
        self.rows, self.kv, self.step, self.causal, self.window, self.ctas = rows, kv_heads, step, causal, window, ctas

    def items(self, n):
        return -(-n // self.step)

    def keys(self, row, q):
        start, n = row
        t = q * self.step
        last = min(t + self.step, n) - 1
        return first_key(start + t, self.window), last_key(start + last, start + n, self.causal, self.window)

    def blocks(self, row, q):
        lo, hi = self.keys(row, q)
        return -(-hi // BLOCK) - lo // BLOCK

    def weigh(self, row):
        return sum(self.blocks(row, q) + COST for q in range(self.items(row[1])))

    def walk(self, cta):
        """[(b, hk, q, first block, last block, part)] of a CTA and what it says of a split item."""
        total = sum(self.weigh(r) for r in self.rows) * self.kv
        quota = max(LEAST, -(-total // self.ctas))
        c0 = quota * cta
        c1 = min(c0 + quota, total)
        got, split = [], None
        if c0 >= c1:
            return got, split
        base = 0
        for b, r in enumerate(self.rows):
            w = self.weigh(r) * self.kv
            if base + w > c0:
                break
            base += w
        weight, x = w // self.kv, base
        hk = (c0 - x) // weight
        x += hk * weight
        q = 0
        while x + self.blocks(r, q) + COST <= c0:
            x += self.blocks(r, q) + COST
            q += 1
        while x < c1:
            n = self.blocks(r, q)
            w = n + COST
            u0, u1 = max(c0 - x, 0) - COST, min(c1 - x, w) - COST
            lo, hi = max(u0, 0), max(u1, 0)
            if hi > lo:
                part = -1 if lo == 0 and hi == n else 1 if lo == 0 else 0
                if part == 1:
                    split = (b, hk, q, (x + w - 1) // quota)
                got.append((b, hk, q, lo, hi, part))
            x += w
            q += 1
            if q == self.items(r[1]):
                q = 0
                hk += 1
                if hk == self.kv:
                    hk = 0
                    b += 1
                    while b < len(self.rows) and self.rows[b][1] == 0:
                        b += 1
                    if b >= len(self.rows):
                        break
                    r = self.rows[b]
        return got, split


@pytest.mark.parametrize("seed", range(300))
def test_every_block_is_taken_once(seed):
    g = random.Random(seed)
    rows = [(g.choice([0, g.randint(0, 5000)]), g.choice([0, 1, g.randint(1, 900)])) for _ in range(g.randint(1, 9))]
    p = Plan(rows, g.choice([1, 2, 5, 8]), g.choice([256, 128, 84, 32, 2]), g.random() < 0.7,
             g.choice([None, None, (0, 0), (40, 0), (700, 64)]), g.choice([148, 148, 3, 1]))
    want = {(b, h, q): p.blocks(r, q) for b, r in enumerate(rows) for h in range(p.kv) for q in range(p.items(r[1]))}
    assert all(n >= 1 for n in want.values())
    taken, walks = {}, [p.walk(c) for c in range(p.ctas)]
    for c, (got, split) in enumerate(walks):
        assert sum(part == 0 for *_, part in got) <= 1 and sum(part == 1 for *_, part in got) <= 1
        assert (split is not None) == any(part == 1 for *_, part in got)
        for k, (b, h, q, lo, hi, part) in enumerate(got):
            assert part != 0 or k == 0  # the rest of an item that began before
            assert part != 1 or k == len(got) - 1
            taken.setdefault((b, h, q), []).append((lo, hi, c, part))
    assert taken.keys() == want.keys()
    for item, parts in taken.items():
        assert parts[0][0] == 0 and parts[-1][1] == want[item]
        assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
        if len(parts) == 1:
            assert parts[0][3] == -1
            continue
        first = parts[0][2]
        assert walks[first][1] == (*item, parts[-1][2])
        assert [c for *_, c, _ in parts] == list(range(first, parts[-1][2] + 1))
        assert [part for *_, part in parts] == [1] + [0] * (len(parts) - 1)


@pytest.mark.parametrize("seed", range(200))
def test_turns_never_arrive_twice(seed):
    """The two tiles' warps on their named barriers, interleaved at random: no barrier is ever
    completed by two arrivals, and both come to the end."""
    g = random.Random(seed)
    items = [g.choice([0, 1, 1, 2, 5]) for _ in range(g.randint(1, 30))]
    arrived, done, blocked = [0, 0], [0, 0], [False, False]

    def ops(i):
        turns = 0
        for n in items:
            for _ in range(n):
                if i == 1 or turns > 0:
                    yield "wait"
                yield "pass"
                turns += 1

    run = [list(ops(0)), list(ops(1))]
    at = [0, 0]
    while at[0] < len(run[0]) or at[1] < len(run[1]):
        able = [i for i in (0, 1) if at[i] < len(run[i]) and (run[i][at[i]] == "pass" or arrived[i] > 0)]
        assert able, "both wait"
        i = g.choice(able)
        if run[i][at[i]] == "wait":
            arrived[i] -= 1
        else:
            arrived[1 - i] += 1
            assert arrived[1 - i] <= 1, "a second arrival before the partner has waited"
        at[i] += 1
