"""The paged cache on the GPU: writing, reading back and attention over the pages against
64 bits, at the sizes, masks and layouts where they can go wrong. Slots that hold no token
are NaN throughout, table entries that mean nothing name no page."""
import math

import pytest
import torch

from svod_b200 import ops
from svod_b200 import _lib as L
from tests.paged_reference import Case, EPS, quantise, stored

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(BF16, False), (BF16, True), (F16, False), (F16, True)]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cache_of(c):
    up = lambda t: None if t is None else t.cuda()
    return ops.PagedCache(up(c.k), up(c.v), up(c.ks), up(c.vs))


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16 if t.element_size() == 2 else torch.int32)


def attend(c, opts=None, cache=None, q=None, lens=True):
    return ops.attention_paged(c.q.cuda() if q is None else q, cache or cache_of(c), c.table.cuda(), i32(c.held),
                               i32(c.new) if lens else None, opts)


def check(got, c, **mask):
    ops.device_status()
    want, lse, bound = c.attention(**mask)
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all()
    worst = (off / bound.clamp(min=2.0 ** -40)).max() if off.numel() else 0.0
    assert worst <= 1.0, float(worst)
    for b, n in enumerate(c.new):
        assert (got[b, n:] == 0).all()
    return lse


# ------------------------------------------------------------------------------ write, read
@pytest.mark.parametrize("dtype,quantized", TYPES + [(F32, False), (F32, True)])
@pytest.mark.parametrize("heads,d,page", [(2, 128, 16), (3, 64, 32), (1, 80, 48), (2, 40, 7), (1, 256, 1), (5, 16, 128),
                                          (1, 13, 5), (2, 512, 8)])
def test_write_is_the_definition(dtype, quantized, heads, d, page):
    c = Case(d + page, 4, 9, [0, 5, page, 3 * page + 1], [9, 0, 4, 1], heads, heads, d, page, dtype, quantized)
    cache = cache_of(c)
    fill = lambda xs: torch.stack([torch.nn.functional.pad(x[h:h + n], (0, 0, 0, 0, 0, 9 - n)) for x, h, n in zip(xs, c.held, c.new)]).cuda()
    ops.cache_write(fill(c.keys), fill(c.values), cache, c.table.cuda(), i32(c.held), i32(c.new))
    ops.device_status()
    c.put(c.held, [h + n for h, n in zip(c.held, c.new)])
    for got, want in ((cache.k, c.k), (cache.v, c.v), (cache.k_scale, c.ks), (cache.v_scale, c.vs)):
        if want is not None:
            assert torch.equal(raw(got.cpu()), raw(want))  # every other slot as it was, to the bit


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_write_8_bits_of_odd_values(dtype):
    """Rows of zeros, of one value, at the borders of a power of two, tiny, huge, with NaN
    and infinities; -0.0 and values that round to the smallest step."""
    d = 64
    top = torch.finfo(dtype).max
    rows = [torch.zeros(d), torch.full((d,), 448.0), torch.full((d,), -449.0 if dtype == F16 else -450.0),
            torch.linspace(-1, 1, d), torch.full((d,), torch.finfo(dtype).tiny), torch.linspace(0, top, d),
            torch.tensor([1.0] * 63 + [math.nan]), torch.tensor([1.0] * 63 + [math.inf]), torch.tensor([-math.inf] + [0.0] * 63),
            torch.tensor([448.0] + [2.0 ** -k for k in range(1, 64)]), torch.tensor([1.75] + [-0.0] * 63),
            torch.tensor([1.7578125] + [0.25] * 63), torch.full((d,), 2.0 ** -24)]
    x = torch.stack(rows).to(dtype).view(1, len(rows), 1, d)
    cache = ops.PagedCache.empty(2, 16, 1, d, dtype, quantized=True)
    ops.cache_write(x.cuda(), x.flip(1).cuda(), cache, i32([[1]]), i32([2]))
    ops.device_status()
    v, e = quantise(x[0, :, 0])
    assert torch.equal(cache.k_scale.cpu()[1, 0, 2:2 + len(rows)].view(torch.uint8).double(), e + 127)
    got = cache.k.cpu()[1, 2:2 + len(rows), 0].double()
    assert torch.equal(got, v)
    assert torch.equal(cache.v.cpu()[1, 2:2 + len(rows), 0].double(), v.flip(0))
    k, _ = ops.cache_read(cache, i32([[1]]), i32([2 + len(rows)]), dtype=dtype)
    want = stored(x[0, :, 0], dtype, True).to(dtype)
    assert torch.equal(k[0, 2:, 0].cpu()[:len(rows)].nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


@pytest.mark.parametrize("dtype,quantized", TYPES + [(F32, False), (F32, True)])
@pytest.mark.parametrize("heads,d,page", [(2, 128, 16), (3, 64, 32), (1, 80, 48), (2, 40, 7), (1, 256, 1), (1, 13, 5)])
def test_read_is_the_definition(dtype, quantized, heads, d, page):
    held = [0, 1, page, 2 * page + 3]
    c = Case(page + d, 4, 1, held, [0] * 4, heads, heads, d, page, dtype, quantized)
    c.put([0] * 4, held)
    length = max(held) + 5
    k, v = ops.cache_read(cache_of(c), c.table.cuda(), i32(held), length, dtype)
    ops.device_status()
    assert k.dtype == dtype and k.shape == (4, length, heads, d)
    for b, n in enumerate(held):
        assert torch.equal(k[b, :n].cpu(), stored(c.keys[b], dtype, quantized).to(dtype))
        assert torch.equal(v[b, :n].cpu(), stored(c.values[b], dtype, quantized).to(dtype))
        assert (k[b, n:] == 0).all() and (v[b, n:] == 0).all()


def test_layers_of_one_buffer_and_views():
    """A layer, a slice of the heads and keys beside values of one buffer; strided new rows."""
    big = torch.full((3, 10, 16, 2, 6, 64), math.nan, dtype=BF16, device="cuda")  # layer, page, slot, k | v, head
    view = ops.PagedCache(big[1, :, :, 0, 2:5], big[1, :, :, 1, 2:5])
    qkv = torch.randn(2, 20, 12 * 64, device="cuda").to(BF16).view(2, 20, 12, 64)
    table = i32([[9, 3, 0, 0, 0, 1], [4, 5, 0, 0, 0, 1]])[:, :2]
    before = big.clone()
    ops.cache_write(qkv[:, :, 6:9], qkv[:, :, 9:12], view, table, i32([1, 0]))
    k, v = ops.cache_read(view, table, i32([21, 20]), 21)
    ops.device_status()
    assert torch.equal(k[1, :20], qkv[1, :, 6:9]) and torch.equal(v[0, 1:], qkv[0, :, 9:12])
    before[1, 9, 1:, :, 2:5] = torch.stack([qkv[0, :15, 6:9], qkv[0, :15, 9:12]], 1)
    before[1, 3, :5, :, 2:5] = torch.stack([qkv[0, 15:, 6:9], qkv[0, 15:, 9:12]], 1)
    before[1, 4, :, :, 2:5] = torch.stack([qkv[1, :16, 6:9], qkv[1, :16, 9:12]], 1)
    before[1, 5, :4, :, 2:5] = torch.stack([qkv[1, 16:, 6:9], qkv[1, 16:, 9:12]], 1)
    assert torch.equal(raw(big), raw(before))
    q = qkv[:, :, :6]
    got = ops.attention_paged(q, view, table, i32([1, 0]), None, ops.Attn(causal=True))
    # row 1 starts its sequence: the framework's contiguous attention says the same
    want = ops.attention(q[1:].contiguous(), qkv[1:, :, 6:9].contiguous(), qkv[1:, :, 9:12].contiguous(), ops.Attn(causal=True))
    assert (got[1:].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


# -------------------------------------------------------------------------------- attention
SHAPES = [
    # heads, kv_heads, d, page
    (4, 2, 128, 16), (2, 2, 64, 32), (6, 2, 64, 64), (8, 1, 128, 128), (3, 1, 96, 48), (4, 4, 40, 8), (2, 1, 128, 256),
    (4, 2, 80, 24), (2, 1, 64, 7), (2, 2, 200, 16), (1, 1, 13, 3), (12, 2, 128, 16),
]


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", SHAPES)
def test_one_token(dtype, quantized, heads, kv, d, page):
    held = [0, 1, page - 1, page, 127, 128, 129, 700]
    c = Case(heads + d, len(held), 1, held, [1, 1, 1, 1, 1, 0, 1, 1], heads, kv, d, page, dtype, quantized)
    c.put([0] * len(held), [h + n for h, n in zip(c.held, c.new)])
    check(attend(c), c)


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", SHAPES)
@pytest.mark.parametrize("tokens", [5, 19])
def test_few_tokens(dtype, quantized, heads, kv, d, page, tokens):
    held, new = [0, 3, 250, 64], [tokens, 2, tokens - 1, 0]
    c = Case(heads + d + tokens, 4, tokens, held, new, heads, kv, d, page, dtype, quantized)
    c.put([0] * 4, [h + n for h, n in zip(held, new)])
    check(attend(c), c)


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", SHAPES[:8])
@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, (40, 0)), (False, (100, 30)), (True, (0, 0))])
def test_chunks(dtype, quantized, heads, kv, d, page, causal, window):
    held, new = [0, 130, 61], [300, 7, 200]
    c = Case(heads + d, 3, 300, held, new, heads, kv, d, page, dtype, quantized)
    c.put([0] * 3, [h + n for h, n in zip(held, new)])
    check(attend(c, ops.Attn(causal=causal, window=window)), c, causal=causal, window=window)


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("tokens", [1, 4, 40])
@pytest.mark.parametrize("window", [(0, 0), (200, 0), (1, 64)])
def test_window_leaves_old_pages_alone(dtype, quantized, tokens, window):
    """Pages that a window has left behind are somebody else's: their entries may be gone
    from the table and nothing of them is looked at."""
    page, held = 16, [900, 333]
    c = Case(3, 2, tokens, held, [tokens, tokens], 4, 2, 128, page, dtype, quantized)
    c.put([max(0, h - window[0]) for h in held], [h + tokens for h in held])
    for b, h in enumerate(held):
        c.table[b, :max(0, h - window[0]) // page] = -1
    check(attend(c, ops.Attn(causal=True, window=window)), c, window=window)


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("tokens", [1, 3, 150])
def test_scale_lse_and_loud_scores(dtype, quantized, tokens):
    held, new = [500, 0], [tokens, max(1, tokens - 1)]
    c = Case(8, 2, tokens, held, new, 4, 2, 64, 32, dtype, quantized, loud=6.0)
    c.put([0, 0], [h + n for h, n in zip(held, new)])
    for scale in (None, 0.7, 0.01):
        o, lse = attend(c, ops.Attn(causal=True, scale=scale, want_lse=True))
        want = check(o, c, scale=scale)
        live = torch.isfinite(want)
        assert torch.equal(torch.isfinite(lse.cpu()), live)
        # scores are sums of D products in 32 bits; their largest is below 64 * 25 here
        assert (lse.cpu().double() - want)[live].abs().max() <= 2.0 ** -24 * 72 * 1600 + 2.0 ** -18


def test_other_scales():
    """Zero and negative scales, which the tensor-core kernels leave to the exact one."""
    c = Case(9, 2, 3, [20, 0], [3, 3], 2, 1, 64, 16, BF16, False)
    c.put([0, 0], [23, 3])
    for scale in (0.0, -0.5):
        check(attend(c, ops.Attn(causal=True, scale=scale)), c, scale=scale)


@pytest.mark.parametrize("quantized", [False, True])
def test_f32(quantized):
    c = Case(5, 2, 17, [30, 0], [17, 9], 4, 2, 72, 16, F32, quantized)
    c.put([0, 0], [47, 9])
    check(attend(c), c)
    check(attend(c, ops.Attn(causal=False)), c, causal=False)


@pytest.mark.parametrize("dtype,quantized", TYPES)
def test_one_heavy_key_among_thousands(dtype, quantized):
    """A key of weight 1 beside 20000 of weight 2^-19 together: what the small ones add up
    to is not lost, whatever the type of the weights in the product."""
    n, d = 20001, 128
    c = Case(1, 1, 1, [n - 1], [1], 2, 1, d, 64, dtype, quantized)
    c.keys[0].zero_()
    c.keys[0][0, 0, 0] = 19 * math.log(2.0) * math.sqrt(d) / 4
    c.q.zero_()
    c.q[..., 0] = 4.0
    c.values[0].fill_(1.0)
    c.values[0][0] = 0.0
    c.put([0], [n])
    check(attend(c), c)


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("tokens", [1, 70])
def test_long_cache(dtype, quantized, tokens):
    held = [9000, 40, 5000]
    c = Case(2, 3, tokens, held, [tokens] * 3, 4, 2, 128, 16, dtype, quantized)
    c.put([0] * 3, [h + tokens for h in held])
    check(attend(c, lens=False), c)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes, the tokens in its last pages."""
    pages, page, h, d = 9000, 256, 8, 128
    c = Case(4, 1, 130, [300], [130], 8, 8, d, page, BF16, False)
    c.put([0], [430])
    big = [torch.empty(pages, page, h, d, dtype=BF16, device="cuda") for _ in "kv"]
    moved = pages - c.pages
    for x, src in zip(big, (c.k, c.v)):
        x[moved:] = src.cuda()
    table = c.table.clone()
    table[0, :2] += moved
    cache = ops.PagedCache(*big)
    got = ops.attention_paged(c.q.cuda(), cache, table.cuda(), i32(c.held))
    check(got, c)
    one = ops.attention_paged(c.q[:, -1:].cuda(), cache, table.cuda(), i32([429]))
    assert (one.double() - got[:, -1:].double()).abs().max() <= 2 * c.attention()[2][:, -1:].max()
    k, _ = ops.cache_read(cache, table.cuda(), i32([430]), 430)
    assert torch.equal(k[0].cpu(), c.keys[0])
    ops.cache_write(k + 1, k, cache, table.cuda(), i32([0]))
    assert torch.equal(big[0][table[0, 0].item()], (k + 1)[0, :256]) and torch.equal(big[1][table[0, 1].item(), :174], k[0, 256:])


# ------------------------------------------------------------------------ bad rows, refusals
@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("tokens", [1, 200])
def test_bad_rows_are_reported(dtype, quantized, tokens):
    """A table entry that names no page, a start below zero, a row that leaves its table:
    the status word says so, rows beside them are what they are, nothing is touched."""
    held = [40, 60, 30, 50]
    c = Case(6, 4, tokens, held, [tokens] * 4, 4, 2, 128, 16, dtype, quantized)
    c.put([0] * 4, [h + tokens for h in held])
    good = attend(c)
    ops.device_status()
    for what in ("entry", "start", "reach"):
        table, start = c.table.clone(), i32(held)
        if what == "entry":
            table[1, 1] = c.pages
        elif what == "start":
            start[1] = -1
        else:
            start[1] = 16 * table.shape[1] - tokens + 1
        cache = cache_of(c)
        got = ops.attention_paged(c.q.cuda(), cache, table.cuda(), start)
        with pytest.raises(ops.OpsError, match="out of range"):
            ops.device_status()
        for b in (0, 2, 3):
            assert torch.equal(got[b], good[b])
        if what != "entry":
            assert (got[1] == 0).all()
            kept = cache_of(c)
            new = torch.ones(4, tokens, 2, 128, dtype=dtype, device="cuda")
            ops.cache_write(new, new, cache, table.cuda(), start)
            with pytest.raises(ops.OpsError, match="out of range"):
                ops.device_status()
            mine = c.table[1, :-(-(held[1] + tokens) // 16)].long()
            assert torch.equal(raw(cache.k)[mine.cuda()], raw(kept.k)[mine.cuda()])
    ops.device_status()


def test_refusals():
    q = torch.zeros(2, 3, 4, 64, dtype=BF16, device="cuda")
    cache = ops.PagedCache.empty(4, 16, 2, 64)
    q8 = ops.PagedCache.empty(4, 16, 2, 64, quantized=True)
    table, start = i32([[0, 1], [2, 3]]), i32([0, 0])
    kv = torch.zeros(2, 3, 2, 64, dtype=BF16, device="cuda")

    def refused(kind, f, *a):
        with pytest.raises(ops.OpsError) as e:
            f(*a)
        assert e.value.kind == kind, e.value

    A = ops.attention_paged
    refused("Shape", A, q[0], cache, table, start)
    refused("Shape", A, q, cache, table[:1], start)
    refused("Shape", A, q, cache, table, start[:1])
    refused("Shape", A, q, cache, table, start, i32([1, 1, 1]))
    refused("Shape", A, q[..., :32], cache, table, start)
    refused("Heads", A, q[:, :, :3], cache, table, start)
    refused("Dtype", A, q.half(), cache, table, start)
    refused("Dtype", A, q, ops.PagedCache(q8.k, q8.v), table, start)
    refused("Dtype", A, q, ops.PagedCache(cache.k, cache.v, q8.k_scale, q8.v_scale), table, start)
    refused("Dtype", A, q, ops.PagedCache(q8.k, q8.v, q8.k_scale.float(), q8.v_scale), table, start)
    refused("Shape", A, q, ops.PagedCache(q8.k, q8.v, q8.k_scale[:3], q8.v_scale), table, start)
    refused("Shape", A, q, ops.PagedCache(cache.k, cache.v[:3]), table, start)
    refused("Unrealized", A, q.cpu(), cache, table, start)
    refused("Unrealized", A, q, cache, table.cpu(), start)
    for opts in (ops.Attn(bias=torch.zeros(2, 4, 3, 32, dtype=BF16, device="cuda")), ops.Attn(chunk=ops.Chunk(4)),
                 ops.Attn(splits=2), ops.Attn(keys=ops.KeyMask.Lens(start)), ops.Attn(seg_start=torch.zeros(2, 3, dtype=torch.int32, device="cuda")),
                 ops.Attn(window=(-1, 0))):
        refused("Graph", A, q, cache, table, start, None, opts)
    W = ops.cache_write
    refused("Shape", W, kv[0], kv[0], cache, table, start)
    refused("Shape", W, kv, kv[:, :2], cache, table, start)
    refused("Shape", W, kv[:, :, :1], kv[:, :, :1], cache, table, start)
    refused("Dtype", W, kv.half(), kv.half(), cache, table, start)
    refused("Launch", W, cache.k[:2, :3], kv, cache, table, start)
    refused("Launch", W, kv, kv, ops.PagedCache(cache.k, cache.k), table, start)
    refused("Graph", W, kv, kv, ops.PagedCache(cache.k[:1].expand(4, -1, -1, -1), cache.v), table, start)
    refused("Unrealized", W, kv.cpu(), kv, cache, table, start)
    R = ops.cache_read
    refused("Shape", R, cache, table, start[:1])
    refused("Dtype", R, cache, table, start, 4, F16)
    refused("Graph", R, q8, table, start, 4, torch.int32)
    ops.device_status()


def test_empty_calls():
    cache = ops.PagedCache.empty(4, 16, 2, 64)
    mk = lambda *s: torch.zeros(*s, dtype=BF16, device="cuda")
    assert ops.attention_paged(mk(0, 3, 4, 64), cache, i32([[]]).view(0, 0), i32([])).shape == (0, 3, 4, 64)
    assert ops.attention_paged(mk(2, 0, 4, 64), cache, i32([[0], [1]]), i32([0, 0])).shape == (2, 0, 4, 64)
    got = ops.attention_paged(mk(2, 3, 4, 64) + 1, cache, i32([[], []]).view(2, 0), i32([0, 0]), i32([0, 0]))
    assert (got == 0).all()
    none = ops.PagedCache.empty(0, 16, 2, 64)
    got = ops.attention_paged(mk(2, 3, 4, 64) + 1, none, i32([[], []]).view(2, 0), i32([0, 0]), i32([0, 0]))
    assert (got == 0).all()
    ops.cache_write(mk(2, 0, 2, 64), mk(2, 0, 2, 64), cache, i32([[0], [1]]), i32([0, 0]))
    k, v = ops.cache_read(cache, i32([[0], [1]]), i32([3, 0]), 0)
    assert k.shape == (2, 0, 2, 64)
    ops.device_status()


# ------------------------------------------------------------------ as they are used together
@pytest.mark.parametrize("dtype,quantized", TYPES)
def test_a_prompt_by_chunks_and_then_token_by_token(dtype, quantized):
    """Write, attend, write, attend: what comes out is the attention of the whole, however
    the sequence was cut."""
    total, cuts = 150, [0, 70, 140, 141, 142, 150]
    c = Case(11, 2, total, [0, 0], [total, total - 8], 8, 2, 64, 16, dtype, quantized)
    cache = cache_of(c)
    pad = torch.nn.functional.pad
    k, v = (torch.stack([pad(x, (0, 0, 0, 0, 0, total - x.shape[0])) for x in xs]).cuda() for xs in (c.keys, c.values))
    q, table, got = c.q.cuda(), c.table.cuda(), []
    for lo, hi in zip(cuts, cuts[1:]):
        start, lens = i32([lo, lo]), i32([hi - lo, max(0, min(hi, total - 8) - lo)])
        ops.cache_write(k[:, lo:hi], v[:, lo:hi], cache, table, start, lens)
        got.append(ops.attention_paged(q[:, lo:hi], cache, table, start, lens))
    check(torch.cat(got, 1), c)
    back, _ = ops.cache_read(cache, table, i32([total, total - 8]), total, dtype)
    for b in range(2):
        assert torch.equal(back[b, :c.new[b]].cpu(), stored(c.keys[b], dtype, quantized).to(dtype))


@pytest.mark.parametrize("quantized", [False, True])
def test_shared_prefix(quantized):
    """Two sequences over the same first pages."""
    c = Case(12, 1, 60, [0], [60], 4, 2, 128, 16, BF16, quantized).put([0], [60])
    cache = cache_of(c)
    table = c.table.cuda().repeat(2, 1)
    table[1, 3] = c.table[0].new_tensor([p for p in range(c.pages) if p not in c.table[0, :4].tolist()])[0].item()
    new = torch.randn(2, 12, 2, 128, device="cuda").to(BF16)
    ops.cache_write(new[1:], new[1:], cache, table[1:], i32([48]))
    a = ops.attention_paged(c.q[:, 48:].cuda().repeat(2, 1, 1, 1), cache, table, i32([48, 48]))
    check(torch.cat([ops.attention_paged(c.q[:, :48].cuda(), cache, table[:1], i32([0])), a[:1]], 1), c)
    d = Case(12, 1, 60, [0], [60], 4, 2, 128, 16, BF16, quantized)
    for xs in (d.keys, d.values):
        xs[0][48:] = new[1].cpu()
    want, _, bound = d.attention()
    assert ((a[1].double().cpu() - want[0, 48:]).abs() <= bound[0, 48:]).all()


@pytest.mark.parametrize("dtype,quantized", TYPES)
def test_graphs_streams_and_repeats(dtype, quantized):
    """Two captured decoding steps replayed at once on two streams, with lengths that move
    on between replays; results are the eager call's to the bit, twice over."""
    made = []
    for seed, tokens in ((21, 1), (22, 90)):
        held = [700, 90, 0, 301]
        c = Case(seed, 4, tokens, held, [tokens] * 4, 8, 2, 128, 16, dtype, quantized)
        c.put([0] * 4, [h + tokens for h in held])
        cache, q, table, start = cache_of(c), c.q.cuda(), c.table.cuda(), i32(held)
        eager = ops.attention_paged(q, cache, table, start)
        short = ops.attention_paged(q, cache, table, start // 2)
        assert torch.equal(eager, ops.attention_paged(q, cache, table, start))
        check(eager, c)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                ops.attention_paged(q, cache, table, start)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = ops.attention_paged(q, cache, table, start)
        made.append((g, s, out, start, eager, short, cache, q, table))  # a graph reads them where they are
    torch.cuda.synchronize()
    for turn in range(3):
        for g, s, *_ in made:
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for _, _, out, start, eager, short, *_ in made:
            assert torch.equal(out, short if turn == 1 else eager)
            out.zero_()
            start.copy_(start // 2) if turn == 0 else start.copy_(i32([700, 90, 0, 301]))
        torch.cuda.synchronize()
    ops.device_status()
    made.clear()


def test_refused_inside_packed_rows():
    lens = i32([40, 64])
    cache = ops.PagedCache.empty(4, 16, 2, 64)
    q = torch.zeros(2, 64, 2, 64, dtype=BF16, device="cuda")
    with ops.PackedRows(lens, 64):
        with pytest.raises(ops.OpsError) as e:
            ops.attention_paged(q, cache, i32([[0], [1]]), i32([0, 0]))
        assert e.value.code == ops.ERR_UNSUPPORTED


# --------------------------------------------------------------- what a caller may also hand over
@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("heads,kv,d,page,tokens", [(2, 1, 128, 8, 1), (2, 1, 128, 8, 70), (96, 1, 64, 16, 1), (128, 1, 128, 32, 3),
                                                    (130, 1, 64, 16, 2), (40, 1, 128, 16, 1), (7, 7, 64, 16, 65), (5, 1, 128, 64, 40)])
def test_wide_groups_and_small_pages(dtype, quantized, heads, kv, d, page, tokens):
    held = [150, 0, 33]
    c = Case(heads + page, 3, tokens, held, [tokens, tokens, max(0, tokens - 1)], heads, kv, d, page, dtype, quantized)
    c.put([0] * 3, [h + n for h, n in zip(held, c.new)])
    check(attend(c), c)


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("batch,tokens", [(75, 1), (75, 40), (1500, 1)])
def test_wide_batches(dtype, quantized, batch, tokens):
    held = [(37 * b) % 260 for b in range(batch)]
    new = [0 if b % 11 == 3 else 1 + b % tokens for b in range(batch)]
    c = Case(batch, batch, tokens, held, new, 2, 1, 64, 16, dtype, quantized)
    c.put([0] * batch, [h + n for h, n in zip(held, new)])
    check(attend(c), c)


@pytest.mark.parametrize("tokens", [3, 90])
@pytest.mark.parametrize("dtype,quantized", TYPES)
def test_what_stands_in_padding_does_not_matter(dtype, quantized, tokens):
    """NaN queries behind the real ones, counts beyond the chunk and below zero, counts and
    tables of 64-bit integers."""
    held = [70, 5, 0]
    c = Case(31, 3, tokens, held, [tokens - 1, tokens, 0], 4, 2, 64, 16, dtype, quantized)
    c.put([0] * 3, [h + n for h, n in zip(held, c.new)])
    q = c.q.cuda()
    q[0, tokens - 1:] = math.nan
    q[2] = math.nan
    lens = torch.tensor([tokens - 1, tokens + 7, -3], device="cuda")
    got = ops.attention_paged(q, cache_of(c), c.table.cuda().long(), torch.tensor(held, device="cuda"), lens)
    c.new = [tokens - 1, tokens, 0]
    c.q[0, tokens - 1:] = 0
    c.q[2] = 0
    check(got, c)


@pytest.mark.parametrize("dtype,quantized", TYPES)
@pytest.mark.parametrize("tokens", [1, 80])
def test_a_row_of_nan_stays_in_its_sequence(dtype, quantized, tokens):
    """A key row that holds a NaN makes NaN of every query that sees it, and of nothing in
    the rows beside it."""
    held = [90, 90]
    c = Case(17, 2, tokens, held, [tokens] * 2, 4, 2, 64, 16, dtype, quantized)
    c.keys[0][20, 1, 3] = math.nan
    c.values[0][20, 1, 3] = math.inf
    c.put([0] * 2, [h + tokens for h in held])
    got = attend(c)
    ops.device_status()
    assert torch.isnan(got[0, :, 2:].float()).all() and torch.isfinite(got[0, :, :2].float()).all()
    want, _, bound = c.attention()
    assert ((got[1].double().cpu() - want[1]).abs() <= bound[1]).all()


def test_reads_past_the_table_are_reported():
    c = Case(3, 2, 1, [20, 9], [0, 0], 1, 1, 64, 16, BF16, False).put([0, 0], [20, 9])
    table = c.table[:, :2].contiguous().cuda()
    k, _ = ops.cache_read(cache_of(c), table, i32([33, 9]), 40)
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    assert (k[0] == 0).all() and torch.equal(k[1, :9].cpu(), c.keys[1])
    k, _ = ops.cache_read(cache_of(c), table, i32([20, -4]), 40)
    ops.device_status()
    assert torch.equal(k[0, :20].cpu(), c.keys[0]) and (k[1] == 0).all()


def test_which_kernel_ran():
    q = torch.randn(2, 40, 4, 64, device="cuda").to(BF16)
    cache, start = ops.PagedCache.empty(12, 16, 2, 64), i32([0, 0])
    table = i32([[0, 1, 2], [3, 4, 5]])
    ops.attention_paged(q, cache, table, start)
    assert ops.chosen().startswith("attention_paged: kernel paged_flash_attention")
    ops.attention_paged(q[:, :5], cache, table, start)
    assert ops.chosen().startswith("attention_paged: kernel paged_decode")
    odd = ops.PagedCache.empty(12, 15, 2, 64)
    ops.attention_paged(q, odd, table, start)
    assert ops.chosen() == "attention_paged: graph shape"
    ops.cache_write(q[:, :, :2], q[:, :, 2:], cache, table, start)
    assert ops.chosen().startswith("cache_write: kernel")
    ops.cache_read(cache, table, start)
    assert ops.chosen().startswith("cache_read: kernel")
    ops.device_status()


def test_launches_are_counted():
    """Two for the 128-row tiles and their merge, one for few rows, one for pages no tile takes."""
    q = torch.randn(2, 40, 4, 64, device="cuda").to(BF16)
    start, table = i32([0, 0]), i32([[0, 1, 2], [3, 4, 5]])
    for page, tokens, want in ((16, 40, 2), (16, 9, 2), (16, 8, 1), (15, 40, 1)):
        cache = ops.PagedCache.empty(12, page, 2, 64)
        for lens in (None, torch.tensor([tokens, 3], device="cuda")):  # the compiled call path and the general one
            before = ops.launches
            ops.attention_paged(q[:, :tokens], cache, table, start, lens)
            assert ops.launches - before == want
    ops.device_status()


@pytest.mark.parametrize("dtype,quantized", TYPES)
def test_two_calls_at_once(dtype, quantized):
    """The tiles, few rows and a read over one cache on three streams side by side, in turns."""
    g = torch.Generator(device="cuda").manual_seed(31)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    cache = ops.PagedCache.empty(200, 16, 2, 128, dtype, quantized)
    table = torch.randperm(200, device="cuda", generator=g).to(torch.int32).view(2, 100)
    ops.cache_write(mk(2, 1600, 2, 128), mk(2, 1600, 2, 128), cache, table, i32([0, 0]))
    chunk, step = mk(2, 300, 8, 128), mk(2, 1, 8, 128)
    calls = [lambda: ops.attention_paged(chunk, cache, table, i32([1300, 700])),
             lambda: ops.attention_paged(step, cache, table, i32([1599, 800])),
             lambda: ops.cache_read(cache, table, i32([1600, 900]), 1600, dtype)[1]]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], [], []]
    for _ in range(20):
        for f, s, out in zip(calls, streams, got):
            with torch.cuda.stream(s):
                out.append(f())
    torch.cuda.synchronize()
    for w, out in zip(want, got):
        assert all(torch.equal(w, x) for x in out)
    ops.device_status()


def test_a_workspace_too_small_is_refused():
    import ctypes as C
    lib = L.load()
    q, cache, table, start = (torch.zeros(1, 70, 2, 64, dtype=BF16, device="cuda"), ops.PagedCache.empty(8, 16, 1, 64),
                              i32([list(range(8))]), i32([0]))
    keep, out = [], torch.empty_like(q)
    c = ops._paged(cache, table, keep)
    qd, sd, od = ops._desc(q), ops._desc(start), ops._desc(out)
    need = lib.svodb_attention_paged_workspace_bytes(C.byref(qd), C.byref(c))
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    o = L.AttnOpts()
    call = lambda: lib.svodb_attention_paged(C.byref(qd), C.byref(c), C.byref(sd), None, C.byref(o), C.byref(od), torch.cuda.current_stream().cuda_stream)
    assert call() == L.ERR_WORKSPACE
    o.workspace, o.workspace_bytes = ws.data_ptr(), need - 1
    assert call() == L.ERR_WORKSPACE
    o.workspace_bytes = need
    assert call() == L.OK
    ops.device_status()


def test_other_python_threads_run_while_a_call_waits(tmp_path):
    """The compiled call path lets the interpreter go around the paged cache's entry points
    (each replaced by one that sleeps), and what torch cannot give is an exception."""
    import ctypes as C
    import subprocess
    import threading
    import time
    (tmp_path / "nap.c").write_text("#include <unistd.h>\nint nap(void) { usleep(400000); return 0; }\nlong none(void) { return 0; }\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(tmp_path / "nap.c"), "-o", str(tmp_path / "nap2.so")], check=True)
    lib = C.CDLL(str(tmp_path / "nap2.so"))
    nap, none = (C.cast(f, C.c_void_p).value for f in (lib.nap, lib.none))
    q, kv = torch.zeros(1, 2, 4, 64, dtype=BF16, device="cuda"), torch.zeros(1, 2, 2, 64, dtype=BF16, device="cuda")
    cache, table, start = ops.PagedCache.empty(4, 16, 2, 64), i32([[0, 1]]), i32([0])
    fast = L.fastops()
    ticks, stop = [0], threading.Event()

    def tick():
        while not stop.wait(0.005):
            ticks[0] += 1

    other = threading.Thread(target=tick)
    other.start()
    try:
        fast.init_paged(nap, nap, nap, none)
        for call in (lambda: fast.cache_write(kv, kv, cache, table, start, None), lambda: fast.cache_read(cache, table, start, 5, BF16),
                     lambda: fast.attention_paged(q, cache, table, start, None, ops.Attn(causal=True))):
            before, t = ticks[0], time.monotonic()
            assert call() is not None and time.monotonic() - t > 0.3
            assert ticks[0] - before > 10
    finally:
        stop.set()
        other.join()
        L._fast = None
        ops._call = None
        L.fastops()  # bound to the library again
    assert ops.attention_paged(q, cache, table, start).shape == q.shape and ops.chosen().startswith("attention_paged")
