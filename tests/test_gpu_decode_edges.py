"""Cached decoding on the GPU where it can go wrong: values that are not finite, far apart or at the end of their type,
calls past 32-bit counts, the larger and smaller head sizes.  Oracle and bounds as in test_gpu_decode.py; each
test derives what it adds.
"""

import numpy as np
import pytest

from hackathon_b200 import rotary
from oracle import decode as O
from test_gpu_decode import HALF_STEP, U, call, close, host, status, tree_inputs, tree_tolerance, values

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


SHAPES = [(1, 4, 1), (5, 4, 1), (10, 8, 1), (40, 8, 1)]  # tokens, q heads, kv heads: 4, 20, 80, 320 rows of a kv head


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("nats", [9, 14, 16, 17])
@pytest.mark.parametrize("cap", [256, 1000])
@pytest.mark.parametrize("T,hq,hk", SHAPES)
def test_tail_far_below_the_largest_scores(t, T, hq, hk, cap, nats, dtype):
    """Every other key `nats` above the rest, with values of 0: tiny weights, alike, on values with a mean are the
    whole output.

    fp16 weights are at least 2**7 where the largest stands, so a weight is off by half a step of its own or, below
    fp16's normal range, by 2**-25: 2**-32 of the largest."""
    n, d = cap - T, 64
    q, k, v = (values(t, dtype, *s, seed=80 + i) for i, s in enumerate([(1, T, hq, d), (1, hk, cap, d), (1, hk, cap, d)]))
    q.zero_()
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[:, :, ::2, 0] = nats                     # 8 * nats / sqrt(64)
    v.mul_(0.25).add_(1.0).mul_(2.0 ** 13)
    v[:, :, ::2] = 0.0
    out = call("tree_attention", [q, k, v, t.tensor([n], dtype=t.int32).cuda(), None], [t.empty_like(q)])[0]
    vv = v[0, 0].double()
    for tok in range(T):
        rows = n + tok + 1
        total = (rows + 1) // 2 * np.exp(float(nats)) + rows // 2
        want = host(vv[:rows].sum(0) / total)
        size = host(vv[:rows].abs().sum(0) / total)
        ulps = 8 * nats + rows + 16            # scores: products of whole numbers, the scale, the base-2 argument; the sums
        half = HALF_STEP[dtype]
        tol = (2 * ulps * U + (0 if dtype == "f32" else half) + POLYNOMIAL) * size + half * np.abs(want)
        if dtype == "fp16":
            tol = tol + rows * 2.0 ** -32 * np.exp(float(nats)) / total * host(vv[:rows].abs().amax(0))
        close(out[0, tok], np.broadcast_to(want, (hq, d)), tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,hq,hk,d", [(1, 1, 1, 64), (1, 4, 1, 128), (2, 4, 1, 256), (3, 4, 1, 64), (5, 4, 1, 128), (20, 20, 1, 64),
                                       (40, 8, 1, 128)])
def test_values_near_the_largest(t, T, hq, hk, d, dtype):
    """Three keys of values 5e37, the later ones 5.4 nats above the first: no sum of weighted values may leave
    the type's range, as none does whose weights are at most 1."""
    n, cap = 250 - T, 250
    q, k, v = (values(t, dtype, *s, seed=90 + i) for i, s in enumerate([(1, T, hq, d), (1, hk, cap, d), (1, hk, cap, d)]))
    q.zero_()
    q[..., 0] = float(d) ** 0.5
    k.zero_()
    k[..., 0] = -100.0
    k[:, :, 0, 0] = 0.0
    for at in (128, 192):
        k[:, :, at, 0] = 5.40625
    v.fill_(5e37)
    out = call("tree_attention", [q, k, v, t.tensor([n], dtype=t.int32).cuda(), None], [t.empty_like(q)])[0]
    want = np.full((1, T, hq, d), float(v[0, 0, 0, 0]))
    # exact weights would leave v itself; what rounding does to them it does above and below the line, the
    # 16-bit kernels' own rounding of a weight excepted
    close(out, want, ((2 * 800 + cap) * U + POLYNOMIAL + 2 * HALF_STEP[dtype]) * want)


@pytest.mark.parametrize("T,hq,d,cap", [(6, 2, 64, 200), (3, 8, 64, 700), (20, 2, 128, 200), (12, 12, 128, 700), (9, 3, 256, 300),
                                        (2, 4, 64, 300), (6, 1, 256, 400)])
def test_fp32_values_at_the_end_of_their_range(t, T, hq, d, cap):
    """The largest finite fp32 values: in a draft that no row sees they leave no trace, in a key against a 0 of the
    query they add 0, in values that are seen they are weighted like others."""
    top = float(np.finfo(np.float32).max)
    q, k, v, lengths, mask = tree_inputs(t, (T, hq, 1, d, cap, [0, 1, cap - T]), "f32", seed=95)
    mask[:, :, 1] = False
    mask[:, 1, 1] = False                      # nobody sees draft 1
    for b, n in enumerate(lengths.tolist()):
        k[b, :, n + 1], v[b, :, n + 1] = -top, -top
        v[b, :, n, 5], v[b, :, n, 6] = -top, top * (1 - 2.0 ** -12)
    q[..., 7] = 0.0
    k[2, :, 0, 7] = top
    out = call("tree_attention", [q, k, v, lengths, t.tensor(mask).cuda()], [t.full_like(q, 7.0)])[0]
    want, size, ulps = O.tree_attention(host(q), host(k), host(v), lengths.tolist(), mask, d ** -0.5)
    # the bound of a score counts |q| |k|, 0 at dim 7; a value cut off keeps 21 bits: 2**-21 of it
    close(out, want, tree_tolerance(want, size, ulps, "f32") + 2.0 ** -21 * size)
    assert status() == 0


def test_rotary_past_32_bit_thread_counts(t):
    """More warps than 2**27: every token is turned, and once."""
    n, d = (1 << 27) + 1000, 4
    x = t.empty(1, n, 1, d, dtype=t.bfloat16, device="cuda").normal_(generator=t.Generator(device="cuda").manual_seed(1))
    pos = t.arange(n, dtype=t.int32, device="cuda")
    steps = rotary.rotary_steps(d, 10000.0)[0]
    places = [slice(0, 1500), slice((1 << 26) - 50, (1 << 26) + 50), slice(n - 1500, n)]
    before = [host(x[:, p]) for p in places]
    call("rotary_embedding", [x, pos, t.tensor(steps).cuda()], [x])  # in place: a token taken twice turns twice
    for p, a in zip(places, before):
        want = O.turned(a, host(pos[p]).astype(np.int64)[None], steps, 1.0, 0)
        close(x[:, p], want, 2.0 ** -20 * O.pair_size(a, d, 1.0, 0) + HALF_STEP["bf16"] * np.abs(want) + 1e-7)


def test_tree_attention_past_32_bit_thread_counts(t):
    """More query rows at one row a joining warp than 2**27 warps: the rows of segments that were cut are all joined."""
    hk, g, d, cap = 130, (1 << 20) - 16, 136, 260
    if t.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB of device memory")
    q = t.zeros(1, 1, hk * g, d, dtype=t.bfloat16, device="cuda")
    k, v = values(t, "bf16", 1, hk, cap, d, seed=1), values(t, "bf16", 1, hk, cap, d, seed=2)
    out = t.full_like(q, 7.0)
    call("tree_attention", [q, k, v, t.tensor([cap - 1], dtype=t.int32).cuda(), None], [out])
    # a query of zeros: equal weights, the mean of the values
    want = v[0].double().mean(1)
    size = v[0].double().abs().mean(1)
    for h in range(hk):
        off = (out[0, 0, h * g:(h + 1) * g].double() - want[h]).abs().amax(0)
        assert (off <= (2.0 ** -16 + 2 * cap * U) * size[h] + HALF_STEP["bf16"] * want[h].abs() + 1e-7).all(), h
    assert status() == 0
    del q, out
    t.cuda.empty_cache()


# tokens, q heads, kv heads, capacity, lengths: 6, 12, 16 and 40 rows of a kv head, cut and uncut, ragged
HEADS = [(2, 6, 2, 900, [898, 0, 131]), (3, 8, 2, 700, [697, 64]), (4, 4, 1, 200, [196, 3]), (10, 4, 1, 600, [590, 255, 1])]


def exact_tolerance(want, size, ulps, dtype, n, v_max):
    """Up to 16 rows (any number at head sizes above 128) 16-bit weights go with what their rounding leaves: off by half a
    step of half a step, in fp16 at least by 2**-32 of the largest weight for each of n keys."""
    weights = 0.0 if dtype == "f32" else HALF_STEP[dtype] ** 2
    err = (2 * ulps * U + weights) * size + (n * 2.0 ** -32 * v_max if dtype == "fp16" else 0.0)
    return (1 + HALF_STEP[dtype]) * err + HALF_STEP[dtype] * np.abs(want) + 1e-7


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("d", [256, 136, 200, 132, 128, 64, 40, 32, 8, 4])
@pytest.mark.parametrize("case", HEADS)
def test_head_sizes(t, case, d, dtype):
    """Boxes wider than a head, heads of up to two 128-dim halves in the kernels and in the join, whole and in part."""
    T, hq, hk, cap, lengths = case
    q, k, v, n, mask = tree_inputs(t, (T, hq, hk, d, cap, lengths), dtype, seed=75)
    out = call("tree_attention", [q, k, v, n, t.tensor(mask).cuda()], [t.full_like(q, 7.0)])[0]
    assert status() == 0
    want, size, ulps = O.tree_attention(host(q), host(k), host(v), lengths, mask, d ** -0.5)
    if T * hq // hk <= 16 or d > 128:
        tol = exact_tolerance(want, size, ulps, dtype, cap, host(v.abs().max()))
    else:
        tol = tree_tolerance(want, size, ulps, dtype) + POLYNOMIAL * size
    close(out, want, tol)


@pytest.mark.parametrize("g", [4, 16, 40])
def test_fp32_sums_over_many_rows_do_not_drift(t, g):
    """Equal weights (queries of zeros) on values with a mean, 40000 rows of 160 heads, so that each block adds up
    thousands of rows.  Roundings to nearest are as often up as down: over 10240 sums their mean is within
    8 sigma = 8 sqrt(additions / 3) u / sqrt(10240); a value itself may lose 2**-21 of it.  Sums that are cut off at every
    addition would all fall short, by 7e-6."""
    hk, n, d = 160, 40_000, 64
    k = t.zeros(1, hk, n + 1, d, device="cuda")
    v = t.empty_like(k).normal_(1.0, 0.25, generator=t.Generator(device="cuda").manual_seed(3))
    q = t.zeros(1, 1, hk * g, d, device="cuda")
    out = call("tree_attention", [q, k, v, t.tensor([n], dtype=t.int32).cuda(), None], [t.empty_like(q)])[0]
    want = t.stack([v[0, h].double().mean(0) for h in range(hk)])
    off = (out.view(hk, g, d).double() / want[:, None] - 1).mean((0, 2)).abs().max().item()
    assert off <= 2.0 ** -21 + 8 * (n / 8 / 3) ** 0.5 * U / (hk * d) ** 0.5
    assert status() == 0
    del k, v, out
    t.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("cap", [250, 700])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,hq,hk", SHAPES)
def test_scores_too_large_for_a_fraction(t, T, hq, hk, d, cap, dtype):
    """Equal scores of 2**33 and more, where fp32's steps are hundreds of powers of two: equal weights all the same, since
    a score less itself is 0."""
    n = cap - T
    q, k, v = (values(t, dtype, *s, seed=100 + i) for i, s in enumerate([(1, T, hq, d), (1, hk, cap, d), (1, hk, cap, d)]))
    q.fill_(1.65625 * (2.0 ** 15 if dtype == "fp16" else 2.0 ** 30))  # no power of two: products with 1 / ln 2 are rounded
    k.fill_(1.71875 * (2.0 ** 15 if dtype == "fp16" else 2.0 ** 30))
    out = call("tree_attention", [q, k, v, t.tensor([n], dtype=t.int32).cuda(), None], [t.empty_like(q)])[0]
    vv = v[0, 0].double()
    for tok in range(T):
        rows = n + tok + 1
        want, size = host(vv[:rows].mean(0)), host(vv[:rows].abs().mean(0))
        half = HALF_STEP[dtype]
        close(out[0, tok], np.broadcast_to(want, (hq, d)), (rows * U + half) * size + half * np.abs(want) + 1e-7)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("base,step", [((4096.0, 4080.0), 7), ((8192.0, 8160.0), 8), ((2048.0, 2040.0), 10)])
@pytest.mark.parametrize("T,hq,hk", SHAPES)
def test_large_scores_a_step_apart(t, T, hq, hk, base, step, dtype):
    """A score of about 2**24 to 2**27 and, units later, one a few nats above it, near where the running maximum is
    raised: no weight leaves the type.  The values of both keys are alike, all others' weights are 0."""
    n, cap, d = 250 - T, 250, 64
    q, k, v = (values(t, dtype, *s, seed=110 + i) for i, s in enumerate([(1, T, hq, d), (1, hk, cap, d), (1, hk, cap, d)]))
    q.zero_()
    k.zero_()
    q[..., 0], q[..., 1] = base[0], 1.0
    for at in (0, 128, 192):
        k[:, :, at, 0], k[:, :, at, 1] = base[1], float(step if at else 0)
        v[:, :, at] = 3.0
    out = call("tree_attention", [q, k, v, t.tensor([n], dtype=t.int32).cuda(), None], [t.empty_like(q)], {"scale": 1.0})[0]
    close(out, np.full((1, T, hq, d), 3.0), (250 * U + 2 * HALF_STEP[dtype]) * 3.0)
