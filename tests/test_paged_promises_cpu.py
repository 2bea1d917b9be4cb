"""What the header and the docstrings promise of the paged cache, where a promise was once more
than the kernels keep."""
import re
from pathlib import Path

import torch

from svod_b200 import ops

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
    for f in sorted(csrc.glob("*.cu*")):
        for line in f.read_text().splitlines():
            if "kStatusBadIndex" in line and "atomicExch" in line:
                assert "status + 1" in line, (f.name, line)
