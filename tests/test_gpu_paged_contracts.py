"""What the paged cache promises beyond its formulas: entries that are no page, slots written
twice, the top of a type's range, integers of 64 bits."""
import math

import pytest
import torch

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
