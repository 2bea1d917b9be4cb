"""What the header and the docstrings promise of the paged cache, where a promise was once more
than the kernels keep."""
import re
from pathlib import Path

from svod_b200 import ops

HEADER = (Path(__file__).resolve().parent.parent / "include" / "svodb.h").read_text()


def words(text):
    return " ".join(re.sub(r"[*`]", " ", text).split())


def test_no_promise_about_a_slot_written_twice():
    """Values and scales of a slot are stores of several threads: neither token is left whole."""
    for text in (words(HEADER), words(ops.cache_write.__doc__)):
        assert "leave either" not in text and "may hold parts of both" in text
