"""Edges of the decoding operators' contracts that need no GPU."""
import os
import re

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "nspeech_b200", "csrc")


@pytest.mark.parametrize("name", ["nq8_beam.cu", "nq8_cache.cu", "nq8_window_attention.cu", "nq8_window_attention.cuh",
                                  "nq8_window_attention_tc.cu"])
def test_decoding_kernels_read_by_plain_loads(name):
    """These kernels start before their predecessor has ended: what it writes must not go through the read-only path."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(r"__ldg|__ldcs|ld\.global\.nc|__restrict__", code)
