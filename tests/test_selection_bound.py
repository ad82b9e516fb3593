"""What the two bf16 terms of a query leave out, against the constant that the selection's error bound allows for it."""

import re
from pathlib import Path

import numpy as np

SOURCE = Path(__file__).resolve().parents[1] / "nano_vllm_jax_b200" / "csrc" / "block_select.cuh"


def _cut(x):
    return (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)


def test_two_terms_of_a_query_leave_no_more_than_the_bound_allows():
    """Every f32 number of one binade (the others are these times a power of two), as two terms that are both cut."""
    allowed = float.fromhex(re.search(r"kSlip = kTerms > 1 \? (0x[0-9a-fp.+-]+)", SOURCE.read_text())[1])
    x = (np.arange(1 << 23, dtype=np.uint32) | np.uint32(0x3F800000)).view(np.float32)
    rest = x - _cut(x)
    rest = rest - _cut(rest)
    largest = (rest.astype(np.float64) / x).max()
    assert largest <= allowed
    assert largest > allowed / 1.02  # (no wider than it has to be)
