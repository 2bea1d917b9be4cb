"""What the header and the docstrings promise of the paged cache, where a promise was once more
than the kernels keep."""
import re
from pathlib import Path

import pytest
import torch

from svod_b200 import _lib as L
from svod_b200 import ops
from tests.test_paged_cache_cpu import error, setup, write

HEADER = (Path(__file__).resolve().parent.parent / "include" / "svodb.h").read_text()


def words(text):
    return " ".join(re.sub(r"[*`]", " ", text).split())


def test_no_promise_about_a_slot_written_twice():
    """Values and scales of a slot are stores of several threads: neither token is left whole."""
    for text in (words(HEADER), words(ops.cache_write.__doc__)):
        assert "leave either" not in text and "may hold parts of both" in text


def test_a_read_with_its_defaults_takes_the_compiled_call_path(monkeypatch):
    asked = []

    class Path:
        def cache_read(self, cache, table, lens, length, dtype):
            asked.append((length, dtype))
            return "k", "v"

    monkeypatch.setattr(ops, "_call", Path())
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for dtype, quantized, want in ((torch.float16, False, torch.float16), (torch.float16, True, torch.bfloat16)):
        cache = ops.PagedCache.empty(4, 16, 2, 64, dtype, quantized, device="cpu")
        assert ops.cache_read(cache, table, lens) == ("k", "v") and asked.pop() == (48, want)
        assert ops.cache_read(cache, table, lens, 5, torch.float32) == ("k", "v") and asked.pop() == (5, torch.float32)


def test_integers_of_64_bits_are_not_cut():
    """A position or a page of 2^32 + 5 is out of range; its low half would be 5."""
    big = torch.tensor([2 ** 32 + 5, -2 ** 40, 7, 2 ** 31, -1])
    want = [2 ** 31 - 1, -2 ** 31, 7, 2 ** 31 - 1, -1]
    assert ops._i32(big).tolist() == want and ops._i32(big).dtype == torch.int32
    assert ops._i32(big.repeat(2, 1).T[:, 0]).tolist() == want
    for dtype in (torch.int8, torch.int16, torch.uint8, torch.int32):
        assert ops._i32(torch.tensor([3, 0, 9], dtype=dtype)).tolist() == [3, 0, 9]
    assert ops._i32(torch.tensor([2 ** 32 - 1], dtype=torch.uint32)).tolist() == [2 ** 31 - 1]
    assert ops._i32(None) is None


def test_an_index_out_of_range_is_no_reason_to_stop_waiting():
    """Waits give up early when their own word is set; the reports of bad indexes go to another."""
    csrc = Path(ops.__file__).resolve().parent / "csrc"
    calls = [(f.name, call) for f in sorted(csrc.glob("*.cu*")) for call in re.findall(r"report_bad_index\(([^)]*)\)", f.read_text())]
    assert len(calls) > 10
    for name, word in calls:
        assert "bad_index" in word or "kBadIndexWord" in word or word == "uint32_t* word", (name, word)
    for f in csrc.glob("*.cu*"):
        stores = [line for line in f.read_text().splitlines() if "kStatusBadIndex" in line and "atomicExch" in line]
        assert f.name == "common.cuh" or not stores


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("apart", [1, 8, 64, 128, 128 * 3 + 64, 128 * 15 + 127, -64, -128 * 7])
def test_keys_and_values_that_share_slots_of_a_page_are_refused(q8, apart):
    """Views of one buffer, some elements apart: [4, 16, 2, 64] pages whose slots are 128 elements."""
    mk, t = setup(q8=q8)
    kind, size = (L.E4M3, 1) if q8 else (L.BF16, 2)
    t["v"] = mk(kind, 4, 16, 2, 64, data=t["k"].data + apart * size)
    k, v, counts = mk(L.BF16, 2, 3, 2, 64), mk(L.BF16, 2, 3, 2, 64), mk(L.I32, 2)
    assert write(t, k, v, counts, None) == L.ERR_ALIAS and "share" in error()


def test_scales_that_share_slots_are_refused():
    mk, t = setup(q8=True)
    t["v_scale"] = mk(L.E8M0, 4, 2, 16, data=t["k_scale"].data + 5)
    assert write(t, mk(L.BF16, 2, 3, 2, 64), mk(L.BF16, 2, 3, 2, 64), mk(L.I32, 2), None) == L.ERR_ALIAS, error()
