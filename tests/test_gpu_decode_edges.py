"""Cached decoding on the GPU where it can go wrong: values that are not finite, far apart or at the end of their type,
calls past 32-bit counts, the larger and smaller head sizes.  Oracle and bounds as in test_gpu_decode.py; each
test derives what it adds.
"""

import numpy as np
import pytest

from oracle import decode as O
from test_gpu_decode import HALF_STEP, U, call, close, host, status, tree_inputs, tree_tolerance

pytestmark = pytest.mark.gpu

POLYNOMIAL = 7.6e-5  # the tcgen05 kernel's exponentials on the FMA pipe, relative


@pytest.fixture(scope="module")
def t():
    import torch
    assert torch.cuda.is_available()
    from hackathon_b200 import _lib
    _lib.lib()
    _lib.device_status()
    return torch


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 96])
@pytest.mark.parametrize("T,hq,hk", [(200, 4, 1), (130, 4, 2), (40, 8, 1), (100, 2, 2)])
def test_infinite_drafts_count_once(t, T, hq, hk, d, dtype):
    """Half of the drafts hold an infinity in dim 3.  Rows that see one are infinite there; every other dim is the plain
    sum, to which each draft's finite values belong once, however many row tiles read them, and call after call."""
    cap = T + 400
    q, k, v, lengths, mask = tree_inputs(t, (T, hq, hk, d, cap, [0, 77, 397]), dtype, seed=70)
    bad = np.zeros((3, T), bool)
    bad[:, ::2] = True
    for b, n in enumerate(lengths.tolist()):
        v[b, :, n:n + T:2, 3] = float("inf")
    d_mask = t.tensor(mask).cuda()
    out = call("tree_attention", [q, k, v, lengths, d_mask], [t.full_like(q, 7.0)])[0]
    for _ in range(20):
        assert t.equal(call("tree_attention", [q, k, v, lengths, d_mask], [t.empty_like(q)])[0], out)
    sees = (mask & bad[:, None, :]).any(-1)
    got = host(out)
    assert np.isposinf(got[sees][..., 3]).all() and np.isfinite(got[~sees][..., 3]).all()
    vv = host(v)
    vv[np.isinf(vv)] = 0
    want, size, ulps = O.tree_attention(host(q), host(k), vv, lengths.tolist(), mask, d ** -0.5)
    rest = np.arange(d) != 3
    tol = tree_tolerance(want, size, ulps, dtype) + POLYNOMIAL * size
    close(out[..., t.tensor(rest).cuda()], want[..., rest], tol[..., rest])
    assert status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("T,hq,d,cap", [(1, 4, 64, 100), (3, 12, 128, 400), (2, 40, 64, 400), (1, 24, 256, 300), (4, 64, 128, 300)])
def test_stale_rows_at_every_offset(t, T, hq, d, cap, dtype):
    """Whatever stands behind the drafts, at each of a unit's rows: the bits of a call with zeros there."""
    lengths = list(range(0, 96, 2)) + list(range(97, 97 - 32, -2))
    q, k, v, n, mask = tree_inputs(t, (T, hq, 2, d, cap, lengths), dtype, seed=71)
    d_mask = t.tensor(mask).cuda()
    behind = (t.arange(cap).cuda() >= n[:, None] + T)[:, None, :, None]
    want = call("tree_attention", [q, k.masked_fill(behind, 0), v.masked_fill(behind, 0), n, d_mask], [t.empty_like(q)])[0]
    assert t.isfinite(want).all()
    for fill in (float("nan"), float("inf")):
        kk, vv = k.masked_fill(behind, fill), v.masked_fill(behind, fill)
        for _ in range(5):
            assert t.equal(call("tree_attention", [q, kk, vv, n, d_mask], [t.empty_like(q)])[0], want)
    assert status() == 0
