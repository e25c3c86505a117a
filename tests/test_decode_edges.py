"""Cached decoding without a GPU: refusals at the ends of the ranges, before any CUDA call."""

import pytest

from hackathon_b200 import _lib as L
from hackathon_b200.kernels import Desc
from test_decode import Space, launch


@pytest.mark.parametrize("capacity", [(1 << 31) - 255, (1 << 31) - 1])
def test_tree_attention_refuses_a_capacity_whose_units_pass_32_bits(capacity):
    """Row counts are rounded up to whole units in 32 bits."""
    gb = 1 << 30
    q, out = Desc(1 * gb, L.BF16, (1, 1, 1, 8)), Desc(2 * gb, L.BF16, (1, 1, 1, 8))
    k, v = Desc(100 * gb, L.BF16, (1, 1, capacity, 8)), Desc(200 * gb, L.BF16, (1, 1, capacity, 8))
    lengths, work = Desc(3 * gb, L.I32, (1,)), Desc(4 * gb, L.U8, (1 << 24,))
    with pytest.raises(RuntimeError, match="capacity"):
        launch("tree_attention", [q, k, v, lengths], [out, work], {})


def test_tree_attention_refuses_heads_of_no_elements():
    n = Space()
    q, k, v, out = (n(L.BF16, *s) for s in ((2, 3, 4, 0), (2, 2, 16, 0), (2, 2, 16, 0), (2, 3, 4, 0)))
    with pytest.raises(RuntimeError, match="head_dim"):
        launch("tree_attention", [q, k, v, n(L.I32, 2)], [out], {})
