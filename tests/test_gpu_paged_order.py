"""Decoding steps of wide batches over pages: more CTAs than the chip holds at once, where rows
are taken longest first. Every row against 64 bits, whatever its place in that order."""
import pytest
import torch

from svod_b200 import ops
from tests.paged_reference import Case

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
TYPES = [(BF16, False), (BF16, True), (F16, False), (F16, True)]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("batch,kv", [(64, 8), (65, 8), (150, 4), (1023, 1), (1024, 1)])
@pytest.mark.parametrize("lengths", ["equal", "ragged", "rising"])
def test_every_row_of_a_wide_batch(dtype, quantized, batch, kv, lengths):
    """Rows of one length, of many (some without a token, one past its table), and longer row by
    row, so that the order turns the batch round; a window in the ragged ones; outputs and lse."""
    d, page = 64, 16
    held = {"equal": [70] * batch, "ragged": [(61 * b) % 400 for b in range(batch)],
            "rising": [2 + 3 * b * 128 // batch for b in range(batch)]}[lengths]
    new = [0 if lengths == "ragged" and b % 13 == 5 else 1 for b in range(batch)]
    window = (300, 0) if lengths == "ragged" else None
    c = Case(batch + kv, batch, 1, held, list(new), kv, kv, d, page, dtype, quantized)
    c.put([0] * batch, [h + n for h, n in zip(held, new)])
    start, bad = i32(held), batch // 2 + 2  # (a row with a token)
    if lengths == "ragged":
        start[bad] = -1
        c.new[bad] = 0
    up = lambda t: None if t is None else t.cuda()
    cache = ops.PagedCache(up(c.k), up(c.v), up(c.ks), up(c.vs))
    got, lse = ops.attention_paged(c.q.cuda(), cache, c.table.cuda(), start, i32(new), ops.Attn(causal=True, window=window, want_lse=True))
    assert "longest_first" in ops.chosen()
    if lengths == "ragged":
        with pytest.raises(ops.OpsError, match="out of range"):
            ops.device_status()
    else:
        ops.device_status()
    want, want_lse, bound = c.attention(window=window)
    assert ((got.double().cpu() - want).abs() <= bound.clamp(min=2.0 ** -40)).all()
    live = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), live) and torch.isneginf(lse.cpu()[~live]).all()
    # scores are sums of 64 products in 32 bits; none is above 64 * 25 / 8 here
    assert (lse.cpu().double() - want_lse)[live].abs().max() <= 2.0 ** -24 * 72 * 200 + 2.0 ** -18


@pytest.mark.parametrize("kv", [1, 8])
@pytest.mark.parametrize("quantized", [False, True])
def test_the_order_costs_no_more_than_the_rows(quantized, kv):
    """1024 short rows, the most that may be put in order, beside 1025, which never are: a CTA's
    share of the order is work in proportion to the batch. (Found by comparing all rows with all
    others, in every CTA, it took several times what the attention did.)"""
    d, page = 128, 64
    cache = ops.PagedCache.empty(64, page, kv, d, BF16, quantized)
    calls = []
    for batch in (1024, 1025):
        q = torch.randn(batch, 1, 2 * kv, d, device="cuda").to(BF16)
        table = (torch.arange(2 * batch, device="cuda", dtype=torch.int32) % 64).view(batch, 2)
        start = torch.arange(batch, device="cuda", dtype=torch.int32) % 127
        calls.append(lambda q=q, table=table, start=start: ops.attention_paged(q, cache, table, start))

    def best(f):
        f()
        took = []
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                f()
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        return min(took)

    ordered, plain = best(calls[0]), best(calls[1])
    ops.device_status()
    assert ordered <= 2 * plain, (ordered, plain)
