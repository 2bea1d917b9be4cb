"""What the paged cache promises beyond its formulas: entries that are no page, slots written
twice, the top of a type's range, integers of 64 bits."""
import math

import pytest
import torch

from svod_b200 import _lib as L
from svod_b200 import ops
from tests.paged_reference import Case

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


@pytest.mark.parametrize("dtype,quantized,page,tokens", [(*t, 16, n) for t in TYPES for n in (1, 90)] + [(*t, 15, 3) for t in TYPES] +
                         [(F32, False, 16, 3), (F32, True, 16, 3)])
def test_an_entry_that_is_no_page_counts_as_zeros(dtype, quantized, page, tokens):
    """In every kernel: keys and values of zeros, with a score of zero, as reading them back gives."""
    held = [70, 40]
    c = Case(page + tokens, 2, tokens, held, [tokens] * 2, 4, 2, 64, page, dtype, quantized)
    c.put([0, 0], [h + tokens for h in held])
    c.table[0, 2] = c.pages + 3
    c.table[1, 0] = -1
    got = ops.attention_paged(c.q.cuda(), cache_of(c), c.table.cuda(), i32(held))
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    for xs in (c.keys, c.values):
        xs[0][2 * page:3 * page] = 0
        xs[1][:page] = 0
    want, _, bound = c.attention()
    assert ((got.double().cpu() - want).abs() <= bound.clamp(min=2.0 ** -40)).all()
    k, _ = ops.cache_read(cache_of(c), c.table.cuda(), i32(held), 70, dtype)
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    assert (k[0, 2 * page:3 * page] == 0).all() and (k[1, :page] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 13])
def test_the_top_of_a_type_reads_back_finite(dtype, d):
    """Values that e4m3 rounds past their type's largest number read back as that number, rows
    that are not finite as NaN."""
    top = torch.finfo(dtype).max
    rows = torch.tensor([1.0, 0.995, 0.96875, 0.9, -1.0, 0.5], dtype=torch.float64) * top
    x = torch.cat([rows[:, None].expand(-1, d), torch.full((1, d), math.inf, dtype=torch.float64)]).to(dtype).view(1, 7, 1, d)
    cache = ops.PagedCache.empty(1, 16, 1, d, dtype, quantized=True)
    ops.cache_write(x.cuda(), -x.cuda(), cache, i32([[0]]), i32([3]))
    k, v = ops.cache_read(cache, i32([[0]]), i32([10]), dtype=dtype)
    ops.device_status()
    for got, want in ((k, x), (v, -x)):
        got = got[0, 3:10, 0].double().cpu()
        assert torch.isnan(got[6]).all()
        assert ((got[:6] - want[0, :6, 0].double()).abs() <= 2.0 ** -4 * want[0, :6, 0].double().abs()).all()
        assert torch.isfinite(got[:6]).all()


@pytest.mark.parametrize("tokens,page", [(1, 16), (8, 16), (90, 16), (3, 15)])
def test_the_top_of_f16_is_finite_in_every_kernel(tokens, page):
    """Keys and values of 65504 in 8-bit pages (256 * 2^8 there): by single tokens, by chunks and
    in the exact kernel."""
    held, d = [150, 37], 64
    c = Case(tokens, 2, tokens, held, [tokens] * 2, 4, 2, d, page, F16, True)
    for ks, vs in zip(c.keys, c.values):
        ks[::5, :, 7] = 65504.0
        ks[1::7, :, 7] = -64000.0
        vs[::3] = 65504.0
        vs[1::9] = -63500.0
    c.q[..., 7] = 2.0 ** -14
    c.put([0, 0], [h + tokens for h in held])
    got = ops.attention_paged(c.q.cuda(), cache_of(c), c.table.cuda(), i32(held))
    ops.device_status()
    assert torch.isfinite(got.float()).all()
    want, _, bound = c.attention()
    # a key's 65536 taken as 65504 moves a score by 32 * 2^-14 / 8, a weight and their sum by as much
    off = 2 * 32 * 2.0 ** -14 / 8 * 65536
    assert ((got.double().cpu() - want).abs() <= bound + off).all()
    one = torch.full_like(c.q[:, -1:], 0)
    for vs in c.values:
        vs[:] = 65504.0
    c.put([0, 0], [h + tokens for h in held])
    got = ops.attention_paged(torch.cat([c.q[:, :-1], one], 1).cuda(), cache_of(c), c.table.cuda(), i32(held))
    assert (got.float() - 65504).abs().max() <= 64


@pytest.mark.parametrize("dtype,quantized", TYPES)
def test_a_slot_written_twice_keeps_to_itself(dtype, quantized):
    """Two rows of one call whose tables name the same page: what its slots hold is nobody's, and
    every other slot is what the call says, to the bit."""
    c = Case(23, 3, 20, [0, 0, 16], [20, 20, 20], 2, 2, 64, 16, dtype, quantized)
    both = c.table[0, 0].item()
    c.table[1, 0] = both
    cache = cache_of(c)
    k, v = (torch.stack([x[h:h + 20] for x, h in zip(xs, c.held)]).cuda() for xs in (c.keys, c.values))
    ops.cache_write(k, v, cache, c.table.cuda(), i32(c.held))
    ops.device_status()
    c.put(c.held, [h + 20 for h in c.held])
    rest = [p for p in range(c.pages) if p != both]
    for got, want in ((cache.k, c.k), (cache.v, c.v), (cache.k_scale, c.ks), (cache.v_scale, c.vs)):
        if want is not None:
            assert torch.equal(raw(got.cpu())[rest], raw(want)[rest])


@pytest.mark.parametrize("tokens", [1, 40])
def test_integers_of_64_bits_that_name_nothing(tokens):
    """A page, a position and a count beyond 32 bits: out of range, not their low halves."""
    held = [30, 20]
    c = Case(5, 2, tokens, held, [tokens] * 2, 4, 2, 64, 16, BF16, False)
    c.put([0, 0], [h + tokens for h in held])
    cache, q, table = cache_of(c), c.q.cuda(), c.table.cuda().long()
    good = ops.attention_paged(q, cache, table, i32(held))
    many = torch.tensor([2 ** 32 + 1, 2 ** 40], device="cuda")  # counts above the chunk's are the chunk's
    assert torch.equal(ops.attention_paged(q, cache, table, i32(held), many), good)
    ops.device_status()
    start = torch.tensor([30, 2 ** 32 + 20], device="cuda")
    got = ops.attention_paged(q, cache, table, start)
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    assert torch.equal(got[0], good[0]) and (got[1] == 0).all()
    table[1, 0] += 2 ** 32
    k, _ = ops.cache_read(cache, table, i32(held), 30)
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    assert (k[1, :16] == 0).all() and torch.equal(k[1, 16:20].cpu(), c.keys[1][16:20])


def test_a_bad_row_does_not_shorten_the_waits_beside_it():
    """A chunk of a million padded tokens, cleared while the row beside the bad one waits for its
    first scores: the same result as behind a short padding."""
    c = Case(41, 2, 200, [0, 3000], [200, 200], 16, 8, 128, 64, BF16, False)
    c.put([0, 0], [200, 3200])
    cache, table, start, lens = cache_of(c), c.table.cuda(), i32([-1, 3000]), i32([200, 200])
    short = ops.attention_paged(c.q.cuda(), cache, table, start, lens)
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    c.new[0] = 0
    want, _, bound = c.attention()
    assert ((short.double().cpu() - want).abs() <= bound.clamp(min=2.0 ** -40)).all()
    q = torch.empty(2, 1 << 20, 16, 128, dtype=BF16, device="cuda")
    q[:, :200] = c.q.cuda()
    for _ in range(2):  # the second call finds the first one's report unread
        got = ops.attention_paged(q, cache, table, start, lens)
        assert torch.equal(got[:, :200], short) and not got[:, 200:].any()
        del got
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    ops.device_status()


def test_one_launch_is_counted_where_the_exact_kernel_takes_the_call():
    q, start, table = torch.randn(2, 40, 4, 64, device="cuda").to(BF16), i32([0, 0]), i32([[0, 1, 2], [3, 4, 5]])
    cache = ops.PagedCache.empty(12, 16, 2, 64)
    for scale, want in ((None, 2), (0.3, 2), (0.0, 1), (-0.5, 1)):
        for lens in (None, torch.tensor([40, 3], device="cuda")):  # the compiled call path and the general one
            before = ops.launches
            ops.attention_paged(q, cache, table, start, lens, ops.Attn(causal=True, scale=scale))
            assert ops.launches - before == want and ops.chosen().startswith("attention_paged: graph") == (want == 1)
    ops.device_status()


def test_a_timeout_is_told_before_a_bad_index():
    cache = ops.PagedCache.empty(2, 16, 1, 64)
    x = torch.zeros(1, 1, 1, 64, dtype=BF16, device="cuda")
    ops.cache_write(x, x, cache, i32([[7]]), i32([0]))
    lib = L.load()
    assert lib.svodb_selftest_wait_timeout(2000, torch.cuda.current_stream().cuda_stream) == L.OK
    with pytest.raises(ops.OpsError, match="wait ran out"):
        ops.device_status()
    ops.device_status()


@pytest.mark.parametrize("dtype,quantized,d", [(*t, 64) for t in TYPES] + [(BF16, True, 13), (F32, False, 64)])
def test_a_cache_without_pages_reports_what_it_cannot_take(dtype, quantized, d):
    cache = ops.PagedCache.empty(0, 16, 2, d, dtype, quantized)
    x, table = torch.ones(2, 3, 2, d, dtype=dtype, device="cuda"), i32([[0, -1], [5, 1]])
    ops.cache_write(x, x, cache, table, i32([0, 7]), i32([0, 0]))
    ops.device_status()
    ops.cache_write(x, x, cache, table, i32([0, 7]))
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    k, v = ops.cache_read(cache, table, i32([3, 10]), 12, dtype)
    with pytest.raises(ops.OpsError, match="out of range"):
        ops.device_status()
    assert not k.any() and not v.any()


@pytest.mark.parametrize("tokens,page", [(1, 16), (70, 16), (3, 15)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_zero_queries_under_a_scale_that_vanishes(dtype, tokens, page):
    """8-bit pages, a query row of zeros and a tiny scale: the row's factor is below 32 bits, every
    key it sees weighs the same and hidden keys weigh nothing."""
    held = [130, 5]
    c = Case(tokens + 1, 2, tokens, held, [tokens] * 2, 4, 2, 64, page, dtype, True)
    c.q[0] = 0
    c.q[1] = c.q[1] * 2.0 ** -14
    c.put([0, 0], [h + tokens for h in held])
    got = ops.attention_paged(c.q.cuda(), cache_of(c), c.table.cuda(), i32(held), None, ops.Attn(causal=True, scale=1e-30))
    ops.device_status()
    want, _, bound = c.attention(scale=1e-30)
    assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("layout", ["pages", "slots", "heads", "columns", "every other page"])
def test_keys_beside_values_in_one_buffer(layout):
    """Views whose spans overlap and whose slots do not are caches."""
    P, S, H, D = 6, 16, 2, 64
    kv = {"pages": lambda b: b.view(P, 2, S, H, D).unbind(1), "slots": lambda b: b.view(P, S, 2, H, D).unbind(2),
          "heads": lambda b: b.view(P, S, H, 2, D).unbind(3), "columns": lambda b: b.view(P, S, H, 2 * D).split(D, -1),
          "every other page": lambda b: (b.view(2 * P, S, H, D)[:-1], b.view(2 * P, S, H, D)[1:])}[layout]
    cache = ops.PagedCache(*kv(torch.full((P * 2 * S * H * D,), math.nan, dtype=BF16, device="cuda")))
    table = i32([[4, 0], [2, 2]])
    x, y, q = (torch.randn(2, 20, h, D, device="cuda").to(BF16) for h in (H, H, 4))
    ops.cache_write(x, y, cache, table, i32([0, 0]), i32([20, 9]))
    k, v = ops.cache_read(cache, table, i32([20, 9]), 20)
    assert torch.equal(k[0], x[0]) and torch.equal(v[0], y[0]) and torch.equal(k[1, :9], x[1, :9]) and torch.equal(v[1, :9], y[1, :9])
    plain = ops.PagedCache(cache.k.contiguous(), cache.v.contiguous())
    for n in (1, 20):
        at = i32([20 - n, 0])
        got = ops.attention_paged(q[:, :n], cache, table, at, i32([n, min(n, 9)]))
        assert torch.isfinite(got.float()).all() and torch.equal(got, ops.attention_paged(q[:, :n], plain, table, at, i32([n, min(n, 9)])))
    ops.device_status()


@pytest.mark.parametrize("tokens", [1, 60])
def test_pages_and_scales_in_records_of_one_buffer(tokens):
    """8-bit keys, values and both scales of a page side by side, as a server's allocator lays them."""
    held, page, h, d = [33, 70], 16, 2, 64
    c = Case(71, 2, tokens, held, [tokens] * 2, 4, h, d, page, F16, True)
    size = page * h * d
    big = torch.full((c.pages, 2 * size + 2 * h * page + 64), 255, dtype=torch.uint8, device="cuda")
    view = lambda lo, n, *s: big[:, lo:lo + n].unflatten(1, s)
    k, v = (view(lo, size, page, h, d).view(torch.float8_e4m3fn) for lo in (0, size))
    ks, vs = (view(2 * size + lo, h * page, h, page).view(torch.float8_e8m0fnu) for lo in (0, h * page))
    cache = ops.PagedCache(k, v, ks, vs)
    total = [n + tokens for n in held]
    pad = lambda xs: torch.stack([torch.nn.functional.pad(x, (0, 0, 0, 0, 0, max(total) - x.shape[0])) for x in xs]).cuda()
    ops.cache_write(pad(c.keys), pad(c.values), cache, c.table.cuda(), i32([0, 0]), i32(total))
    got = ops.attention_paged(c.q.cuda(), cache, c.table.cuda(), i32(held))
    ops.device_status()
    want, _, bound = c.attention()
    assert ((got.double().cpu() - want).abs() <= bound).all()
    assert (big[:, 2 * size + 2 * h * page:] == 255).all()
