"""Lengths as columns of a wider table, and one length for all rows: the ops take them as they would
a contiguous vector."""
import pytest
import torch

from svod_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("layout", ["column", "expanded"])
def test_lengths_of_any_stride(kind, layout):
    plain = torch.tensor([40, 7, 23] if layout == "column" else [31, 31, 31], dtype=kind, device="cuda")
    lens = (torch.stack([plain, plain.new_full((3,), 64)], 1)[:, 0] if layout == "column" else plain[:1].expand(3))
    assert not lens.is_contiguous()
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(3, 64, 2, 64, device="cuda", generator=g).bfloat16() for _ in range(3))
    hidden = torch.randn(3, 64, 128, device="cuda", generator=g).bfloat16()
    at = lambda l: ops.attention(q, k, v, ops.Attn(keys=ops.KeyMask.Lens(l)))
    assert torch.equal(at(lens), at(plain))
    for f in (lambda l: ops.pool(hidden, l, ops.POOL_LAST), lambda l: ops.norm_pool(hidden, aux=l, mode=ops.POOL_LAST)):
        assert torch.equal(f(lens), f(plain))
    ops.device_status()


def test_a_strided_norm_weight_is_refused():
    x, w = torch.randn(4, 64, device="cuda").bfloat16(), torch.randn(128, device="cuda").bfloat16()
    with pytest.raises(ops.OpsError) as e:
        ops.rms_norm(x, w[::2])
    assert e.value.kind == "Shape"
    with pytest.raises(ops.OpsError) as e:
        ops.linear(x, torch.randn(32, 64, device="cuda").bfloat16(), ops.Linear(bias=w[::4]))
    assert e.value.kind == "Shape"
