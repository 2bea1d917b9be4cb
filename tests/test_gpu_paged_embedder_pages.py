"""`Qwen3Embedder.extend` against the stack in 64 bits over the keys and values that its pages hold:
what is left is the roundings of the stream, tight enough to tell 8-bit pages from 16-bit ones."""
import math

import numpy as np
import pytest
import torch

from svod_b200 import ops
from tests import test_gpu_paged_embedder as T
from tests.paged_reference import stored

pytestmark = pytest.mark.gpu

# A layer rounds to bf16 nine times on the way to its output (normed input, query, its rotation's
# table, rotated query, weights, attention, sum, gate and normed sum, sum), each by half a step at
# most: evenly spread errors, 2^-8 / sqrt(3) of the rounded thing's norm. An attention's output is up to
# 1.08 of the stream it joins here. They are independent, so their squares add up.
TOL = 1.1 * math.sqrt(9 * T.LAYERS) * 2.0 ** -8 / math.sqrt(3.0)


def stack64(p, ids, pages=None):
    """(embedding, [(k, v)] of the layers) of one row in 64 bits, attending over `pages` [(k, v)]
    [n, HKV, HD] a layer where given, else over its own keys and values as bf16 holds them."""
    H, HKV, HD, F, cfg = T.H, T.HKV, T.HD, T.F, T.CFG
    t = lambda x: torch.from_numpy(np.asarray(x, dtype=np.float64))
    rms = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * t(w)
    n = len(ids)
    ang = torch.arange(n).double()[:, None] * cfg.rope_theta ** (-torch.arange(0, HD, 2).double() / HD)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    turn = lambda x: torch.cat([x[..., :HD // 2] * cos - x[..., HD // 2:] * sin, x[..., :HD // 2] * sin + x[..., HD // 2:] * cos], -1)
    x, made = t(p["embed"])[torch.as_tensor(ids)], []
    for i, lp in enumerate(p["layers"]):
        qkv = (rms(x, lp["in_w"]) @ t(lp["qkv_w"]).T).view(n, H + 2 * HKV, HD)
        q, k, v = turn(rms(qkv[:, :H], lp["qn_w"])), turn(rms(qkv[:, H:H + HKV], lp["kn_w"])), qkv[:, H + HKV:]
        made.append((k, v))
        k, v = pages[i] if pages is not None else (y.to(torch.bfloat16).double() for y in (k, v))
        k, v = (y.repeat_interleave(H // HKV, 1) for y in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) / HD ** 0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -torch.inf)
        x = x + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(n, H * HD) @ t(lp["o_w"]).T
        g = rms(x, lp["post_w"]) @ t(lp["gu_w"]).T
        x = x + (torch.nn.functional.silu(g[:, :F]) * g[:, F:]) @ t(lp["down_w"]).T
    y = rms(x[-1], p["norm_w"])
    return y / y.norm(), made


@pytest.mark.parametrize("quantized", [False, True])
def test_a_shared_instruction_and_chunks_over_the_pages_they_wrote(quantized):
    """Rows behind a shared instruction, one of them continued by a chunk and by tokens: the pages
    hold the stack's keys and values, and the embedding is the stack's over those pages."""
    p, rng, page = T.weights(), np.random.default_rng(17), 16
    m = T.model(p)
    caches = m.paged_caches(16, page, quantized)
    said, tails = rng.integers(0, T.V, 32), [rng.integers(0, T.V, n) for n in (5, 40, 23)]
    m.extend(T.i32(said[None]), caches, T.i32([[7, 3]]), T.i32([0]))
    table = T.i32([[7, 3, 0, 1, 2], [7, 3, 4, 5, 6], [7, 3, 8, 9, 10]])
    ids = np.zeros((3, 40), dtype=np.int64)
    for r, q in enumerate(tails):
        ids[r, :len(q)] = q
    got = list(m.extend(T.i32(ids), caches, table, T.i32([32] * 3), T.i32([len(q) for q in tails])))
    for more in (rng.integers(0, T.V, 18), rng.integers(0, T.V, 1), rng.integers(0, T.V, 1)):
        got[0] = m.extend(T.i32(more[None]), caches, table[:1], T.i32([32 + len(tails[0])]))[0]
        tails[0] = np.concatenate([tails[0], more])
    ops.device_status()
    for r, q in enumerate(tails):
        row = np.concatenate([said, q])
        held = [tuple(y[0].double().cpu() for y in ops.cache_read(c, table[r:r + 1], T.i32([len(row)]), len(row), torch.bfloat16)) for c in caches]
        want, made = stack64(p, row, held)
        for pages, own in zip(held, made):
            for have, true in zip(pages, own):
                # the stream's error, and what the pages' type rounds
                off = TOL + (2.0 ** -4 if quantized else 2.0 ** -8)
                assert ((have - true).norm(dim=-1) <= off * true.norm(dim=-1)).all()
                if quantized:  # values that e4m3 beside a power of two holds
                    assert torch.equal(stored(have, torch.bfloat16, True), have)
        assert (got[r].double().cpu() - want).norm() <= TOL
        plain, _ = stack64(p, row)
        if quantized:
            assert (plain - want).norm() >= 2 * TOL  # so the bound above tells the pages apart
        else:
            assert (plain - want).norm() <= TOL


def test_chunks_are_slices_of_a_documents_ids():
    p, rng = T.weights(), np.random.default_rng(19)
    m = T.model(p)
    ids, table = T.i32(rng.integers(0, T.V, (2, 90))), T.i32([[0, 1], [3, 2]])
    whole = m.extend(ids, m.paged_caches(4, 64), table, T.i32([0, 0]))
    for kind in (torch.int32, torch.int64):
        caches = m.paged_caches(4, 64)
        for lo, hi in ((0, 50), (50, 89), (89, 90)):
            got = m.extend(ids.to(kind)[:, lo:hi], caches, table, T.i32([lo, lo]))
        ops.device_status()
        assert ((got - whole).double().norm(dim=-1) <= 2 * TOL).all()
