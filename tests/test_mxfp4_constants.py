"""Limits that two files hold are the same in both."""

import re
from pathlib import Path

from titan_amd import mxfp4

CSRC = Path(__file__).resolve().parent.parent / "titan_amd" / "csrc"


def _constant(path, name):
    m = re.search(rf"\b{name} = (\d+)", (CSRC / path).read_text())
    assert m, (path, name)
    return int(m.group(1))


def test_rows_of_the_kernel_for_few():
    assert _constant("torch/binding.cpp", "kFewRows") == _constant("mxfp4_rows.h", "kFewRows")


def test_rows_that_are_sorted():
    assert _constant("torch/binding.cpp", "kSortedMinRows") == mxfp4.SORTED_MIN_ROWS
