"""Embedding over a paged cache (`Qwen3Embedder.extend`): by chunks, behind a shared
instruction, over 16- and 8-bit pages, against the stack in 64 bits with keys and values
stored as the pages store them."""
import numpy as np
import pytest
import torch

from oracle import svod_oracle as O
from svod_b200 import encoders as E
from svod_b200 import ops
from tests.paged_reference import stored

pytestmark = pytest.mark.gpu

V, D, H, HKV, HD, F, LAYERS = 300, 256, 4, 2, 128, 384, 2
CFG = E.Qwen3Config(vocab_size=V, hidden_size=D, num_hidden_layers=LAYERS, num_attention_heads=H, num_key_value_heads=HKV,
                    head_dim=HD, intermediate_size=F)
TOL = 2e-2  # of a unit-norm row against 64 bits: the whole stack's tolerance (see the full-size tests)


def weights():
    rng = np.random.default_rng(42)
    w = lambda shape, sigma=0.02, mean=0.0: O.round_to(O.BF16, rng.standard_normal(shape) * sigma + mean)
    layers = [dict(in_w=w((D,), 0.02, 1.0), qkv_w=w(((H + 2 * HKV) * HD, D), 0.06), qn_w=w((HD,), 0.02, 1.0), kn_w=w((HD,), 0.02, 1.0),
                   o_w=w((D, H * HD), 0.06), post_w=w((D,), 0.02, 1.0), gu_w=w((2 * F, D)), down_w=w((D, F))) for _ in range(LAYERS)]
    return dict(embed=w((V, D), 0.5), layers=layers, norm_w=w((D,), 0.02, 1.0))


def model(p):
    dev = lambda x: torch.from_numpy(np.asarray(x, dtype=np.float32)).to(torch.bfloat16).cuda()
    return E.Qwen3Embedder(CFG, dict(embed=dev(p["embed"]), norm_w=dev(p["norm_w"]),
                                     layers=[{k: dev(v) for k, v in lp.items()} for lp in p["layers"]]))


def embed64(p, ids, quantized):
    """The embedding of one row of ids, keys and values as the pages hold them."""
    t = lambda x: torch.from_numpy(np.asarray(x, dtype=np.float64))
    rms = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + CFG.rms_norm_eps) * t(w)
    n = len(ids)
    ang = torch.arange(n).double()[:, None] * CFG.rope_theta ** (-torch.arange(0, HD, 2).double() / HD)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    turn = lambda x: torch.cat([x[..., :HD // 2] * cos - x[..., HD // 2:] * sin, x[..., :HD // 2] * sin + x[..., HD // 2:] * cos], -1)
    x = t(p["embed"])[torch.as_tensor(ids)]
    for lp in p["layers"]:
        qkv = (rms(x, lp["in_w"]) @ t(lp["qkv_w"]).T).view(n, H + 2 * HKV, HD)
        q, k, v = turn(rms(qkv[:, :H], lp["qn_w"])), turn(rms(qkv[:, H:H + HKV], lp["kn_w"])), qkv[:, H + HKV:]
        k, v = (stored(y.to(torch.bfloat16), torch.bfloat16, quantized).repeat_interleave(H // HKV, 1) for y in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) / HD ** 0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -torch.inf)
        x = x + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(n, H * HD) @ t(lp["o_w"]).T
        g = rms(x, lp["post_w"]) @ t(lp["gu_w"]).T
        x = x + (torch.nn.functional.silu(g[:, :F]) * g[:, F:]) @ t(lp["down_w"]).T
    y = rms(x[-1], p["norm_w"])
    return y / y.norm()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("quantized", [False, True])
def test_queries_behind_a_shared_instruction(quantized):
    """The instruction's pages are written once; three queries of unequal length follow it,
    then one of them grows token by token."""
    p, rng, page = weights(), np.random.default_rng(7), 16
    m = model(p)
    caches = m.paged_caches(16, page, quantized)
    said = rng.integers(0, V, 32)
    queries = [rng.integers(0, V, n) for n in (5, 40, 23)]
    first = m.extend(i32(said[None]), caches, i32([[7, 3]]), i32([0]))
    assert (first[0].double().cpu() - embed64(p, said, quantized)).abs().max() < TOL
    table = i32([[7, 3, 0, 1, 2], [7, 3, 4, 5, 6], [7, 3, 8, 9, 10]])
    ids = np.zeros((3, 40), dtype=np.int64)
    for r, q in enumerate(queries):
        ids[r, :len(q)] = q
    got = m.extend(i32(ids), caches, table, i32([32] * 3), i32([len(q) for q in queries]))
    ops.device_status()
    for r, q in enumerate(queries):
        assert (got[r].double().cpu() - embed64(p, np.concatenate([said, q]), quantized)).abs().max() < TOL
    tail = queries[0]
    for _ in range(3):
        new = rng.integers(0, V, 1)
        got = m.extend(i32(new[None]), caches, table[:1], i32([32 + len(tail)]))
        tail = np.concatenate([tail, new])
        assert (got[0].double().cpu() - embed64(p, np.concatenate([said, tail]), quantized)).abs().max() < TOL
    ops.device_status()


def test_a_document_by_chunks_is_the_document():
    p, rng = weights(), np.random.default_rng(8)
    m = model(p)
    ids = rng.integers(0, V, (2, 300))
    lengths = [300, 211]
    whole = m.forward(i32(ids), i32(lengths))
    caches = m.paged_caches(2 * 5, 64)
    table, rows = i32([[4, 2, 0, 6, 8], [1, 3, 5, 7, 9]]), [None, None]
    for lo, hi in ((0, 128), (128, 211), (211, 300)):
        live = [r for r in (0, 1) if lengths[r] > lo]
        got = m.extend(i32(ids[live, lo:hi]), caches, table[live].contiguous(), i32([lo] * len(live)))
        for r, y in zip(live, got):
            rows[r] = y
    ops.device_status()
    for r in (0, 1):
        want = embed64(p, ids[r, :lengths[r]], False)
        assert (rows[r].double().cpu() - want).abs().max() < TOL
        assert (whole[r].double().cpu() - want).abs().max() < TOL


def test_a_captured_step_moves_on():
    """One captured call, replayed with ids and positions that a user writes into its buffers."""
    p, rng = weights(), np.random.default_rng(9)
    m = model(p)
    ids = rng.integers(0, V, 12)
    eager = m.paged_caches(2, 16)
    table, want = i32([[1, 0]]), []
    for t in range(12):
        want.append(m.extend(i32(ids[None, t:t + 1]), eager, table, i32([t])))
    caches = m.paged_caches(2, 16)
    tok, start = i32([[0]]), i32([0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.extend(tok, caches, table, start)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = m.extend(tok, caches, table, start)
    for t in range(12):
        tok.fill_(int(ids[t])), start.fill_(t)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[t])
    ops.device_status()
    del g


def test_counts_of_any_integer_type_and_stride():
    """`start` and `lens` as columns of a wider table of 64-bit integers."""
    p, rng = weights(), np.random.default_rng(11)
    m = model(p)
    ids = i32(rng.integers(0, V, (3, 20)))
    table = i32([[0, 1], [2, 3], [4, 5]])
    meta = torch.tensor([[0, 20], [0, 7], [0, 13]], device="cuda")
    want = m.extend(ids, m.paged_caches(6, 16), table, i32([0, 0, 0]), i32([20, 7, 13]))
    got = m.extend(ids, m.paged_caches(6, 16), table, meta[:, 0], meta[:, 1])
    meta32 = meta.to(torch.int32)
    narrow = m.extend(ids, m.paged_caches(6, 16), table, meta32[:, 0], meta32[:, 1])
    ops.device_status()
    assert torch.equal(got, want) and torch.equal(narrow, want)
