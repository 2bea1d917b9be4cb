"""Vectors that kernels read element after element (biases, norm weights, lengths, row maps): one
with another stride is refused before anything is launched."""
import ctypes as C

import pytest

from svod_b200 import _lib as L
from tests.test_paged_cache_cpu import Buffers, P, error


def ptr(t):
    return C.pointer(t)


@pytest.mark.parametrize("stride", [0, 2, 7])
def test_a_strided_vector_is_refused(stride):
    lib, mk = L.load(), Buffers()
    vec = lambda dtype, n: mk(dtype, n, strides=(stride,))
    x, w, y = mk(L.BF16, 2, 4, 64), mk(L.BF16, 96, 64), mk(L.BF16, 2, 4, 96)
    o = L.LinearOpts()
    o.bias = ptr(vec(L.BF16, 96))
    assert lib.svodb_linear(P(x), P(w), C.byref(o), P(y), None) == L.ERR_SHAPE and "bias" in error()
    out, good = mk(L.BF16, 2, 4, 64), mk(L.BF16, 64)
    for wt, b in ((vec(L.BF16, 64), None), (good, vec(L.BF16, 64))):
        assert lib.svodb_layer_norm(P(x), P(wt), P(b), 1e-5, P(out), None) == L.ERR_SHAPE, error()
    q, k = mk(L.BF16, 3, 4, 2, 64), mk(L.BF16, 3, 8, 2, 64)
    a = L.AttnOpts()
    a.key_lens = ptr(vec(L.I32, 3))
    assert lib.svodb_attention(P(q), P(k), P(mk(L.BF16, 3, 8, 2, 64)), C.byref(a), P(mk(L.BF16, 3, 4, 2, 64)), None) == L.ERR_SHAPE, error()
    a = L.AttnOpts()
    a.has_cache, a.cache_kv_heads, a.cache_row_map = 1, 2, ptr(vec(L.I32, 3))
    assert lib.svodb_attention(P(q), P(k), P(mk(L.BF16, 3, 8, 2, 64)), C.byref(a), P(mk(L.BF16, 3, 4, 2, 64)), None) == L.ERR_SHAPE, error()
    h = L.QkvOpts()
    h.heads, h.kv_heads, h.head_dim, h.q_norm = 2, 1, 64, ptr(vec(L.BF16, 64))
    outs = [mk(L.BF16, 2, 4, n, 64) for n in (2, 1, 1)]
    assert lib.svodb_heads(P(mk(L.BF16, 2, 4, 256)), C.byref(h), *map(P, outs), None) == L.ERR_SHAPE and "q norm" in error(), error()
    hidden, pooled = mk(L.BF16, 3, 8, 64), mk(L.F32, 3, 64)
    assert lib.svodb_norm_pool(P(hidden), None, None, 1e-5, 1, None, P(vec(L.I32, 3)), 2, 1, P(pooled), None) == L.ERR_SHAPE, error()
