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


class Array:
    """A device array of another library: a description only."""

    def __init__(self, typestr, *shape, at=1 << 20):
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (at, False), "strides": None, "version": 3}

    def reshape(self, *shape):
        return self

    def __getitem__(self, at):
        return self


def test_bool_arrays_are_masks_only(monkeypatch):
    """Kernels that compute on bytes could put a 2 into a bool array: only the mask may be one."""
    from hackathon_b200 import kernel_registry as R
    launched = []
    monkeypatch.setattr(R.L, "launch", lambda kid, *a: launched.append(kid))  # the addresses are made up
    b, f = Array("|b1", 4, 4), Array("<f4", 4, 4, at=2 << 20)
    for name, ins, outs in (("add", [b, b], [b]), ("add", [f, f], [b]), ("relu", [b], [b]), ("transpose", [b], [b])):
        with pytest.raises(TypeError, match="dtype"):
            R.lookup(name)(ins, outs, {})
    q, k, v, o = (Array("<f4", *s, at=i << 20) for i, s in
                  enumerate(((1, 4, 2, 8), (1, 2, 16, 8), (1, 2, 16, 8), (1, 4, 2, 8)), 3))
    lengths = Array("<i4", 1, at=8 << 20)
    with pytest.raises(TypeError, match="dtype"):
        R.lookup("tree_attention")([q, k, v, Array("|b1", 1), b], [o], {})
    with pytest.raises(TypeError, match="dtype"):
        R.lookup("rotary_embedding")([b, lengths, lengths], [b], {})
    assert not launched
    R.lookup("tree_attention")([q, k, v, lengths, b], [o], {})
    assert launched == [L.K_TREE_ATTN]


def test_bool_tensors_are_masks_only():
    torch = pytest.importorskip("torch")
    from hackathon_b200 import kernel_registry as R

    class Fake:  # a torch tensor on a GPU, as far as it is described
        is_cuda, dtype, shape = True, torch.bool, (4, 4)
        is_contiguous = staticmethod(lambda: True)
        data_ptr = staticmethod(lambda: 1 << 20)

    Fake.__module__ = "torch.fake"
    with pytest.raises(TypeError, match="dtype"):
        R.describe(Fake())
    assert R.describe(Fake(), mask=True).dtype == L.U8
