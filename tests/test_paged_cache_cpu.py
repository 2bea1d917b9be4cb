"""The paged cache on the host: what its entry points refuse before anything is launched
(descriptors of buffers that nobody reads), and the 64-bit reference's own roundings."""
import ctypes as C
import math

import pytest
import torch

from svod_b200 import _lib as L
from svod_b200 import ops
from tests.paged_reference import quantise, stored, to_e4m3

BASE = 1 << 40  # never followed: every call here is refused


class Buffers:
    """Descriptors of contiguous tensors, each in an address range of its own."""

    def __init__(self):
        self.at, self.keep = BASE, []

    def __call__(self, dtype, *shape, strides=None, data=None):
        t = L.Tensor()
        t.data = self.at if data is None else data
        self.at += 1 << 32
        t.dtype, t.rank = dtype, len(shape)
        step = 1
        for i in reversed(range(len(shape))):
            t.shape[i], t.stride[i] = shape[i], step
            step *= max(shape[i], 1)
        for i, s in enumerate(strides or ()):
            t.stride[i] = s
        self.keep.append(t)
        return t


def setup(q8=False, pages=4, page=16, heads=2, d=64, batch=2, width=2):
    mk = Buffers()
    t = dict(k=mk(L.E4M3 if q8 else L.BF16, pages, page, heads, d), v=mk(L.E4M3 if q8 else L.BF16, pages, page, heads, d),
             table=mk(L.I32, batch, width))
    if q8:
        t["k_scale"], t["v_scale"] = mk(L.E8M0, pages, heads, page), mk(L.E8M0, pages, heads, page)
    return mk, t


def cache_of(t):
    c = L.PagedCache()
    for n, x in t.items():
        setattr(c, n, C.pointer(x))
    return c


P = lambda t: None if t is None else C.byref(t)


def attention(t, q, start, lens, opts=None, o=None, mk=None):
    lib = L.load()
    o = o or mk(q.dtype, *[q.shape[i] for i in range(q.rank)])
    return lib.svodb_attention_paged(P(q), C.byref(cache_of(t)), P(start), P(lens), C.byref(opts or L.AttnOpts()), P(o), None)


def write(t, k, v, start, lens):
    return L.load().svodb_cache_write(P(k), P(v), C.byref(cache_of(t)), P(start), P(lens), None)


def read(t, lens, k, v):
    return L.load().svodb_cache_read(C.byref(cache_of(t)), P(lens), P(k), P(v), None)


def error():
    return L.load().svodb_last_error().decode()


CACHES = [
    ("k", lambda mk: mk(L.BF16, 4, 16, 128), L.ERR_SHAPE), ("k", lambda mk: mk(L.BF16, 4, 0, 2, 64), L.ERR_SHAPE),
    ("v", lambda mk: mk(L.BF16, 3, 16, 2, 64), L.ERR_SHAPE), ("v", lambda mk: mk(L.F16, 4, 16, 2, 64), L.ERR_DTYPE),
    ("k", lambda mk: mk(L.I32, 4, 16, 2, 64), L.ERR_DTYPE), ("v", lambda mk: mk(L.BF16, 4, 16, 2, 64, strides=(1, 1, 1, 2)), L.ERR_GRAPH),
    ("k", lambda mk: mk(L.BF16, 4, 16, 2, 64, strides=(2048, 128, -64, 1)), L.ERR_GRAPH),
    ("k", lambda mk: mk(L.BF16, 4, 16, 2, 64, data=0), L.ERR_UNREALIZED),
    ("table", lambda mk: mk(L.I32, 3, 2), L.ERR_SHAPE), ("table", lambda mk: mk(L.I32, 4), L.ERR_SHAPE),
    ("table", lambda mk: mk(L.I64, 2, 2), L.ERR_DTYPE), ("table", lambda mk: mk(L.I32, 2, 2, strides=(1, 2)), L.ERR_GRAPH),
    ("table", lambda mk: mk(L.I32, 2, 1 << 27), L.ERR_SHAPE),
    ("k_scale", lambda mk: mk(L.E8M0, 4, 2, 16), L.ERR_DTYPE),
]


@pytest.mark.parametrize("name,make,code", CACHES)
def test_caches_that_every_entry_point_refuses(name, make, code):
    mk, t = setup()
    t[name] = make(mk)
    q, kv, counts = mk(L.BF16, 2, 3, 4, 64), [mk(L.BF16, 2, 3, 2, 64) for _ in "kv"], mk(L.I32, 2)
    assert attention(t, q, counts, None, mk=mk) == code, error()
    assert write(t, *kv, counts, None) == code, error()
    assert read(t, counts, *kv) == code, error()


@pytest.mark.parametrize("name,make,code", [
    ("k_scale", lambda mk: mk(L.U8, 4, 2, 16), L.ERR_DTYPE), ("v_scale", lambda mk: mk(L.E8M0, 4, 16, 2), L.ERR_SHAPE),
    ("v_scale", lambda mk: mk(L.E8M0, 4, 2, 16, strides=(32, 1, 2)), L.ERR_GRAPH), ("v", lambda mk: mk(L.BF16, 4, 16, 2, 64), L.ERR_DTYPE),
])
def test_scales_that_are_refused(name, make, code):
    mk, t = setup(q8=True)
    t[name] = make(mk)
    assert attention(t, mk(L.BF16, 2, 3, 4, 64), mk(L.I32, 2), None, mk=mk) == code, error()
    del t[name if name.endswith("scale") else "v_scale"]
    assert write(t, mk(L.BF16, 2, 3, 2, 64), mk(L.BF16, 2, 3, 2, 64), mk(L.I32, 2), None) == L.ERR_DTYPE, error()


def test_operands_that_are_refused():
    mk, t = setup()
    q, counts = mk(L.BF16, 2, 3, 4, 64), mk(L.I32, 2)
    for bad, code in ((mk(L.BF16, 2, 3, 256), L.ERR_SHAPE), (mk(L.BF16, 2, 3, 4, 32), L.ERR_SHAPE), (mk(L.F16, 2, 3, 4, 64), L.ERR_DTYPE),
                      (mk(L.BF16, 2, 3, 3, 64), L.ERR_HEADS), (mk(L.BF16, 3, 3, 4, 64), L.ERR_SHAPE),
                      (mk(L.BF16, 2, 3, 4, 64, strides=(768, 256, 1, 4)), L.ERR_GRAPH)):
        assert attention(t, bad, counts, None, mk=mk) == code, error()
    for bad, code in ((mk(L.I32, 3), L.ERR_SHAPE), (mk(L.I32, 2, 1), L.ERR_SHAPE), (mk(L.I64, 2), L.ERR_DTYPE),
                      (mk(L.I32, 2, strides=(2,)), L.ERR_GRAPH), (mk(L.I32, 2, data=0), L.ERR_UNREALIZED)):
        assert attention(t, q, bad, None, mk=mk) == code, error()
        assert attention(t, q, counts, bad, mk=mk) == code, error()
    assert attention(t, q, None, None, mk=mk) == L.ERR_UNREALIZED
    for bad, code in ((mk(L.BF16, 2, 3, 4, 32), L.ERR_SHAPE), (mk(L.F16, 2, 3, 4, 64), L.ERR_DTYPE),
                      (mk(L.BF16, 2, 3, 4, 64, strides=(0, 256, 64, 1)), L.ERR_GRAPH), (mk(L.BF16, 2, 3, 4, 64, data=q.data + 64), L.ERR_ALIAS),
                      (mk(L.BF16, 2, 3, 4, 64, data=t["v"].data), L.ERR_ALIAS)):
        assert attention(t, q, counts, None, o=bad) == code, error()
    wide = mk(L.BF16, 2, 3, 4, 320)
    t["k"], t["v"] = mk(L.BF16, 4, 16, 2, 320), mk(L.BF16, 4, 16, 2, 320)
    assert attention(t, wide, counts, None, mk=mk) == L.ERR_UNSUPPORTED, error()


def test_options_that_are_refused():
    mk, t = setup()
    q, counts = mk(L.BF16, 2, 3, 4, 64), mk(L.I32, 2)

    def opts(**kw):
        o = L.AttnOpts()
        for n, x in kw.items():
            setattr(o, n, C.pointer(x) if isinstance(x, L.Tensor) else x)
        return o

    bias, lens, seg = mk(L.BF16, 2, 4, 3, 32), mk(L.I32, 2), mk(L.I32, 2, 3)
    for o, code in ((opts(bias=bias), L.ERR_UNSUPPORTED), (opts(key_lens=lens), L.ERR_UNSUPPORTED), (opts(seg_start=seg), L.ERR_UNSUPPORTED),
                    (opts(has_chunk=1, chunk_size=4), L.ERR_UNSUPPORTED), (opts(has_cache=1), L.ERR_UNSUPPORTED), (opts(splits=2), L.ERR_UNSUPPORTED),
                    (opts(has_window=1, window_left=-1), L.ERR_GRAPH), (opts(lse=mk(L.F32, 2, 3, 4)), L.ERR_SHAPE),
                    (opts(lse=mk(L.BF16, 2, 4, 3)), L.ERR_DTYPE), (opts(lse=mk(L.F32, 2, 4, 3, data=q.data)), L.ERR_ALIAS)):
        assert attention(t, q, counts, None, opts=o, mk=mk) == code, error()


def test_writes_and_reads_that_are_refused():
    mk, t = setup()
    k, v, counts = mk(L.BF16, 2, 3, 2, 64), mk(L.BF16, 2, 3, 2, 64), mk(L.I32, 2)
    for bad, code in ((mk(L.BF16, 2, 3, 128), L.ERR_SHAPE), (mk(L.BF16, 2, 4, 2, 64), L.ERR_SHAPE), (mk(L.BF16, 2, 3, 1, 64), L.ERR_SHAPE),
                      (mk(L.F16, 2, 3, 2, 64), L.ERR_DTYPE), (mk(L.BF16, 2, 3, 2, 64, data=t["k"].data), L.ERR_ALIAS)):
        assert write(t, k, bad, counts, None) == code, error()
    assert read(t, counts, k, mk(L.BF16, 2, 4, 2, 64)) == L.ERR_SHAPE
    assert read(t, counts, k, mk(L.BF16, 2, 3, 2, 64, data=k.data)) == L.ERR_ALIAS
    assert read(t, counts, mk(L.BF16, 2, 3, 2, 64, data=t["v"].data), v) == L.ERR_ALIAS
    assert read(t, counts, mk(L.BF16, 2, 3, 2, 64, strides=(384, 0, 64, 1)), v) == L.ERR_GRAPH
    assert read(t, counts, mk(L.F32, 2, 3, 2, 64), mk(L.F32, 2, 3, 2, 64)) == L.ERR_DTYPE
    t["v"] = t["k"]
    assert write(t, k, v, counts, None) == L.ERR_ALIAS
    mk, t = setup()
    t["k"] = mk(L.BF16, 4, 16, 2, 64, strides=(0, 128, 64, 1))
    assert write(t, k, v, counts, None) == L.ERR_GRAPH, error()
    t["k"] = mk(L.BF16, 4, 16, 2, 64, strides=(2048, 64, 64, 1))
    assert write(t, k, v, counts, None) == L.ERR_GRAPH, error()


def test_the_op_layer_refuses_host_tensors():
    c = ops.PagedCache.empty(4, 16, 2, 64, device="cpu")
    t, q, kv = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3, 4, 64).bfloat16(), torch.zeros(2, 3, 2, 64).bfloat16()
    for call in (lambda: ops.attention_paged(q, c, t, t[0]), lambda: ops.cache_write(kv, kv, c, t, t[0]), lambda: ops.cache_read(c, t, t[0])):
        with pytest.raises(ops.OpsError) as e:
            call()
        assert e.value.kind == "Unrealized"


def test_the_reference_rounds_as_the_type_does():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)]
    assert torch.equal(to_e4m3(every), every)
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(20000, generator=g, dtype=torch.float64) * s for s in (200.0, 1.0, 0.01, 0.001)]).clamp(-448, 448)
    x = torch.cat([x.float().double(), (every.unique()[1:] + every.unique()[:-1]) / 2])
    assert torch.equal(to_e4m3(x), x.float().to(torch.float8_e4m3fn).double())


def test_the_reference_scales_leave_nothing_out():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(500, 64, generator=g) * torch.exp2(torch.randint(-30, 30, (500, 1), generator=g).float())).bfloat16()
    v, e = quantise(x)
    assert (v.abs() <= 448).all() and (v.abs().amax(-1) > 223).all()
    off = (stored(x, torch.bfloat16, True) - x.double()).abs()
    step = torch.exp2(e)[:, None]
    assert (off <= torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)).all()
    assert quantise(torch.zeros(1, 8))[1].item() == -127 and quantise(torch.tensor([[1.0, math.nan]]))[1].item() == 128


def test_boxes_never_straddle_pages():
    """A kernel takes a block of 128 (or 64) keys as boxes of gcd(page_size, block) keys."""
    for page in range(8, 520, 8):
        for block in (64, 128):
            box = math.gcd(page, block)
            assert box >= 8 and block // box <= 16
            for j in range(0, 4 * page * block // box, box):
                assert j // page == (j + box - 1) // page
