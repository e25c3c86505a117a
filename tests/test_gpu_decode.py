"""Cached decoding on the GPU against float64 definitions (oracle/decode.py).

Tolerances, derived before the first run.  u = 2**-24 is half a step of fp32; a 16-bit output is
rounded once, half a step of its type: eps / 2 of the value.

* Rotation: the phase reaches sincospif as a float in [-1, 1] half turns (u relative, times pi), with
  2**-32 turns cut off; sincospif is within 2 ulp; two products, one sum, the scale: below
  (pi + 4 + 4) u < 12 u < 2**-20 of scale * (|a| + |b|).
* Norm: at most D + 8 roundings in the sum of squares, halved by the root, rsqrtf within 2 ulp, two
  products: (D / 2 + 8) u; with D <= 512 below 264 u < 2**-15.9.  The rotation of the normed pair adds its own.
* Attention: a score is off by at most (D + 4) u sum |q k| scale; with e that bound, weights are off by
  2 e relative, sums by a u for each row.  16-bit kernels round each weight to the type as well
  (eps / 2 of it).
"""

import numpy as np
import pytest

from hackathon_b200 import rotary
from oracle import decode as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {"f32": U, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


@pytest.fixture(scope="module")
def t():
    import torch
    assert torch.cuda.is_available()
    from hackathon_b200 import _lib
    _lib.lib()
    _lib.device_status()
    return torch


def types(t):
    return {"f32": t.float32, "bf16": t.bfloat16, "fp16": t.float16}


def status():
    from hackathon_b200 import _lib
    return _lib.device_status()


def call(name, ins, outs, params=None):
    from hackathon_b200.kernel_registry import lookup
    lookup(name)(ins, outs, params or {})
    return outs


def values(t, dtype, *shape, seed=0, at=0):
    """Normal values; `at`: that many elements into a larger buffer, so the pointer is less aligned."""
    g = t.Generator(device="cuda").manual_seed(seed)
    n = int(np.prod(shape))
    buf = t.randn(n + at, generator=g, device="cuda").to(types(t)[dtype])
    return buf[at:].view(*shape)


def host(x):
    return x.detach().double().cpu().numpy()


def close(got, want, tolerance):
    got = host(got)
    assert np.all(np.isfinite(got))
    over = np.abs(got - want) - tolerance
    assert over.max() <= 0, f"{over.max()} over its tolerance at {np.unravel_index(over.argmax(), over.shape)}"


# ------------------------------------------------------------------ rotation

ROTARY = [  # batch, tokens, heads, dim, rotary, elements off alignment
    (2, 5, 4, 64, 64, 0), (1, 1, 1, 2, 2, 0), (3, 7, 5, 80, 20, 0), (1, 33, 3, 96, 48, 0), (2, 3, 7, 128, 64, 0),
    (1, 300, 32, 128, 128, 0), (2, 2, 3, 256, 256, 0), (1, 9, 2, 256, 64, 0), (1, 4, 3, 50, 10, 0), (1, 3, 2, 512, 512, 0),
    (1, 3, 2, 520, 260, 0), (2, 5, 4, 64, 64, 1), (2, 5, 4, 64, 64, 4), (1, 5, 3, 64, 32, 2), (4096, 1, 3, 64, 64, 0),
    (1, 6, 300, 64, 64, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("case", ROTARY)
def test_rotary(t, case, interleaved, dtype):
    b, s, h, d, r, at = case
    x = values(t, dtype, b, s, h, d, seed=1, at=at)
    steps = rotary.rotary_steps(r, 10000.0)[0]
    pos = np.random.default_rng(2).integers(0, 1 << 20, (b, s))
    out = values(t, dtype, b, s, h, d, seed=3, at=at)
    outs = call("rotary_embedding", [x, t.tensor(pos).cuda(), t.tensor(steps).cuda()], [out],
                {"interleaved": interleaved, "scale": 1.25})
    want = O.turned(host(x), pos, steps, 1.25, interleaved)
    tol = 2.0 ** -20 * O.pair_size(host(x), r, 1.25, interleaved) + HALF_STEP[dtype] * np.abs(want) + 1e-7
    tol[..., r:] = 0  # untouched behind the rotated part
    close(outs[0], want, tol)
    # the same in place
    same = x.clone() if not at else x
    outs2 = call("rotary_embedding", [same, t.tensor(pos).cuda(), t.tensor(steps).cuda()], [same],
                 {"interleaved": interleaved, "scale": 1.25})
    assert t.equal(outs2[0], outs[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,r", [(64, 64), (64, 16), (96, 48), (128, 128), (256, 128)])
@pytest.mark.parametrize("heads", [1, 2, 3, 4, 5, 7, 9, 13, 15])
def test_rotary_of_few_heads(t, heads, d, r, dtype):
    """Blocks whose heads begin and end within a token, and whose tokens are of several sequences."""
    for interleaved, (b, s) in enumerate([(13, 29), (5, 1)]):
        x = values(t, dtype, b, s, heads, d, seed=heads)
        steps = rotary.rotary_steps(r, 10000.0)[0]
        pos = np.random.default_rng(heads).integers(0, 1 << 20, (b, s))
        out = call("rotary_embedding", [x, t.tensor(pos).cuda(), t.tensor(steps).cuda()], [t.empty_like(x)],
                   {"interleaved": interleaved, "scale": 0.75})[0]
        want = O.turned(host(x), pos, steps, 0.75, interleaved)
        tol = 2.0 ** -20 * O.pair_size(host(x), r, 0.75, interleaved) + HALF_STEP[dtype] * np.abs(want) + 1e-7
        tol[..., r:] = 0
        close(out, want, tol)


def test_rotary_positions(t):
    """Shared, 32-bit, negative and very far positions; a zero position leaves x as it is."""
    x = values(t, "f32", 3, 4, 2, 64, seed=4)
    steps = rotary.rotary_steps(64, 500000.0, "turns", 8.0)[0]
    d_steps = t.tensor(steps).cuda()
    for pos in (np.array([0, 5, -7, 1 << 30]), np.array([-(1 << 31), (1 << 31) - 1, 1, 2])):
        want = O.turned(host(x), np.broadcast_to(pos, (3, 4)).copy(), steps, 1.0, 0)
        tol = 2.0 ** -20 * O.pair_size(host(x), 64, 1.0, 0)
        for kind in (t.int32, t.int64):
            close(call("rotary_embedding", [x, t.tensor(pos, dtype=kind).cuda(), d_steps], [t.empty_like(x)])[0], want, tol)
    far = np.array([[1 << 40, (1 << 62) + 3, -(1 << 50), 0]] * 3)
    got = call("rotary_embedding", [x, t.tensor(far).cuda(), d_steps], [t.empty_like(x)])[0]
    close(got, O.turned(host(x), far, steps, 1.0, 0), 2.0 ** -20 * O.pair_size(host(x), 64, 1.0, 0))
    assert t.equal(got[:, 3], x[:, 3])


# ------------------------------------------------------------------ norms and rotation

NORM = [  # batch, tokens, q heads, kv heads, dim, rotary, per-head weights, elements off alignment
    (2, 5, 4, 4, 64, 64, 0, 0), (1, 1, 32, 8, 128, 128, 1, 0), (3, 2, 3, 1, 80, 40, 0, 0), (1, 17, 7, 7, 96, 24, 1, 0),
    (2, 3, 8, 2, 256, 64, 0, 0), (1, 4, 2, 1, 20, 20, 1, 0), (1, 2, 2, 2, 512, 256, 0, 0), (2, 3, 2, 1, 64, 64, 1, 1),
    (70, 30, 12, 2, 128, 64, 0, 0), (1, 3, 4, 0, 64, 64, 0, 0),
]


def norm_inputs(t, case, dtype, scale=1.0):
    b, s, hq, hk, d, r, per_head, at = case
    qkv = values(t, dtype, b, s, hq + 2 * hk, d, seed=5, at=at)
    qkv *= scale
    qw = values(t, "f32", hq, d, seed=6) if per_head else values(t, "f32", d, seed=6)
    kw = values(t, "f32", hk, d, seed=7) if per_head else values(t, "f32", d, seed=7)
    steps, factor = rotary.rotary_steps(r, 10000.0, "turns", 2.0)
    pos = np.random.default_rng(8).integers(0, 100000, (b, s))
    return qkv, qw, kw, pos, steps, factor


def norm_want(t, case, qkv, qw, kw, pos, steps, factor, interleaved, dtype, eps=1e-6):
    """q, k, v as they should be, with their tolerances."""
    b, s, hq, hk, d, r, _, _ = case
    x = host(qkv)
    got = []
    for part, w in ((x[:, :, :hq], qw), (x[:, :, hq:hq + hk], kw)):
        n = O.normed(part, None if w is None else host(w), eps)
        want = O.turned(n, pos, steps, factor, interleaved)
        size = O.pair_size(n, r, factor, interleaved)
        got.append((want, ((d / 2 + 8) * U + 2.0 ** -20) * size + HALF_STEP[dtype] * np.abs(want) + 1e-7))
    return got + [(x[:, :, hq + hk:], 0.0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("case", NORM)
def test_qk_norm_rotary(t, case, interleaved, dtype):
    b, s, hq, hk, d, r, _, at = case
    qkv, qw, kw, pos, steps, factor = norm_inputs(t, case, dtype)
    params = {"num_heads": hq, "kv_num_heads": hk, "interleaved": interleaved, "scale": factor}
    ins = [qkv, qw, kw, t.tensor(pos).cuda(), t.tensor(steps).cuda()]
    out = call("qk_norm_rotary", ins, [values(t, dtype, *qkv.shape, seed=9, at=at)], params)[0]
    want = norm_want(t, case, qkv, qw, kw, pos, steps, factor, interleaved, dtype)
    for (w, tol), lo, hi in zip(want, (0, hq, hq + hk), (hq, hq + hk, hq + 2 * hk)):
        if hi > lo:
            close(out[:, :, lo:hi], w, tol)
    flat = qkv.clone().view(b, s, -1)
    same = call("qk_norm_rotary", [flat] + ins[1:], [flat], params)[0]
    assert same.shape == flat.shape
    # in place: the same bits, unless the copy is better aligned and takes wider pieces, which sum in another order
    if not at:
        assert t.equal(same.view_as(out), out)
    for (w, tol), lo, hi in zip(want, (0, hq, hq + hk), (hq, hq + hk, hq + 2 * hk)):
        if hi > lo:
            close(same.view_as(out)[:, :, lo:hi], w, tol)


def test_qk_norm_without_weights_and_without_norm(t):
    case = (2, 5, 4, 2, 64, 32, 0, 0)
    qkv, _, kw, pos, steps, factor = norm_inputs(t, case, "f32")
    d_pos, d_steps = t.tensor(pos).cuda(), t.tensor(steps).cuda()
    heads = {"num_heads": 4, "kv_num_heads": 2, "scale": factor}
    out = call("qk_norm_rotary", [qkv, None, kw, d_pos, d_steps], [t.empty_like(qkv)], heads)[0]
    want = norm_want(t, case, qkv, None, kw, pos, steps, factor, 0, "f32")
    close(out[:, :, :4], *want[0])
    close(out[:, :, 4:6], *want[1])
    out = call("qk_norm_rotary", [qkv, None, None, d_pos, d_steps], [t.empty_like(qkv)], {**heads, "normalize": 0})[0]
    close(out[:, :, :6], O.turned(host(qkv)[:, :, :6], pos, steps, factor, 0),
          2.0 ** -20 * O.pair_size(host(qkv)[:, :, :6], 32, factor, 0))
    assert t.equal(out[:, :, 6:], qkv[:, :, 6:])


def test_qk_norm_of_zero_and_small_heads(t):
    """A zero head stays zero (epsilon keeps it finite), a tiny one is scaled by about 1 / sqrt(eps)."""
    case = (1, 3, 2, 1, 64, 64, 0, 0)
    qkv, qw, kw, pos, steps, factor = norm_inputs(t, case, "f32", scale=1e-5)
    qkv[:, 1] = 0
    out = call("qk_norm_rotary", [qkv, qw, kw, t.tensor(pos).cuda(), t.tensor(steps).cuda()], [t.empty_like(qkv)],
               {"num_heads": 2, "kv_num_heads": 1, "scale": factor, "epsilon": 1e-6})[0]
    want = norm_want(t, case, qkv, qw, kw, pos, steps, factor, 0, "f32")
    close(out[:, :, :2], *want[0])
    assert not out[:, 1].any()


APPEND = [  # case as above, capacity, lengths
    ((2, 1, 4, 4, 64, 64, 0, 0), 9, [0, 8]), ((3, 5, 32, 8, 128, 128, 1, 0), 40, [0, 17, 35]),
    ((2, 7, 3, 1, 80, 20, 0, 0), 7, [0, 0]), ((1, 63, 2, 2, 64, 32, 0, 0), 1000, [501]),
    ((2, 3, 4, 2, 50, 10, 1, 1), 11, [3, 8]), ((3, 21, 2, 1, 64, 64, 0, 0), 60, [0, 11, 39]),
    ((5, 9, 2, 2, 64, 64, 0, 0), 20, [0, 1, 11, 3, 7]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("case,cap,lengths", APPEND)
def test_append(t, case, cap, lengths, interleaved, dtype):
    b, s, hq, hk, d, r, _, at = case
    qkv, qw, kw, pos, steps, factor = norm_inputs(t, case, dtype)
    kc, vc = values(t, dtype, b, hk, cap, d, seed=10, at=at), values(t, dtype, b, hk, cap, d, seed=11, at=at)
    k0, v0 = kc.clone(), vc.clone()
    q, k1, v1 = call("qk_norm_rotary_append",
                     [qkv, qw, kw, t.tensor(pos).cuda(), t.tensor(steps).cuda(), t.tensor(lengths, dtype=t.int32).cuda()],
                     [values(t, dtype, b, s, hq, d, seed=12, at=at), kc, vc],
                     {"num_heads": hq, "kv_num_heads": hk, "interleaved": interleaved, "scale": factor})
    assert k1.data_ptr() == kc.data_ptr() and status() == 0
    want = norm_want(t, case, qkv, qw, kw, pos, steps, factor, interleaved, dtype)
    close(q, *want[0])
    for i, n in enumerate(lengths):
        close(kc[i, :, n:n + s].transpose(0, 1), want[1][0][i], want[1][1][i])
        assert t.equal(vc[i, :, n:n + s].transpose(0, 1), qkv[i, :, hq + hk:])
        for now, before in ((kc, k0), (vc, v0)):  # every other row as it was
            assert t.equal(now[i, :, :n], before[i, :, :n]) and t.equal(now[i, :, n + s:], before[i, :, n + s:])


def test_append_leaves_out_a_sequence_that_does_not_fit(t):
    case = (4, 3, 2, 1, 64, 64, 0, 0)
    qkv, qw, kw, pos, steps, factor = norm_inputs(t, case, "bf16")
    kc, vc = values(t, "bf16", 4, 1, 8, 64, seed=1), values(t, "bf16", 4, 1, 8, 64, seed=2)
    k0, v0 = kc.clone(), vc.clone()
    lengths = t.tensor([5, 6, -1, 2147483647], dtype=t.int32).cuda()
    q = call("qk_norm_rotary_append", [qkv, qw, kw, t.tensor(pos).cuda(), t.tensor(steps).cuda(), lengths],
             [t.zeros(4, 3, 2, 64, dtype=t.bfloat16, device="cuda"), kc, vc],
             {"num_heads": 2, "kv_num_heads": 1, "scale": factor})[0]
    assert status() == 40 and status() == 0
    close(q, *norm_want(t, case, qkv, qw, kw, pos, steps, factor, 0, "bf16")[0])
    assert t.equal(kc[1:], k0[1:]) and t.equal(vc[1:], v0[1:]) and not t.equal(kc[0], k0[0])


# ------------------------------------------------------------------ attention

TREE = [  # tokens, q heads, kv heads, dim, capacity, lengths
    (1, 16, 16, 64, 131, [130]), (1, 1, 1, 64, 1, [0]), (1, 8, 2, 128, 700, [0, 1, 63, 64, 65, 699]),
    (5, 4, 4, 64, 300, [0, 7, 123, 290]), (26, 32, 8, 128, 600, [0, 500, 574]), (64, 14, 2, 128, 200, [0, 63, 136]),
    (17, 7, 1, 64, 90, [73, 5]), (33, 24, 3, 64, 1100, [1031, 1067, 0]), (3, 6, 3, 96, 50, [47, 12]), (2, 2, 1, 256, 77, [75]),
    (4, 3, 3, 80, 20, [16, 0]), (2, 4, 2, 17, 30, [28, 3]), (130, 8, 8, 64, 400, [200]), (300, 2, 1, 128, 333, [33, 0]),
    (1, 64, 1, 128, 5000, [4999]), (8, 16, 1, 128, 700, [692, 5]), (16, 16, 2, 128, 1300, [1284, 127, 128, 129]),
    (7, 40, 1, 64, 2200, [2193, 0]), (11, 12, 1, 96, 900, [889]), (20, 16, 2, 120, 600, [300, 580]), (9, 128, 1, 64, 257, [240, 248]), (1, 5, 5, 1, 9, [8]),
]


def tree_inputs(t, case, dtype, seed=20):
    T, hq, hk, d, cap, lengths = case
    b = len(lengths)
    q, k, v = (values(t, dtype, *s, seed=seed + i) for i, s in
               enumerate([(b, T, hq, d), (b, hk, cap, d), (b, hk, cap, d)]))
    rs = np.random.RandomState(seed)
    mask = np.zeros((b, T, T), bool)
    for i in range(T):  # random trees
        if i:
            parent = rs.randint(max(0, i - 6), i, b)
            mask[:, i] = mask[np.arange(b), parent]
        mask[:, i, i] = True
    return q, k, v, t.tensor(lengths, dtype=t.int32).cuda(), mask


def tree_tolerance(out, size, ulps, dtype):
    weights = 0.0 if dtype == "f32" else HALF_STEP[dtype]
    return (2 * ulps * U + weights) * size + HALF_STEP[dtype] * np.abs(out) + 1e-7


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("kind", ["tree", "shared", "chain"])
@pytest.mark.parametrize("case", TREE)
def test_tree_attention(t, case, kind, dtype):
    q, k, v, lengths, mask = tree_inputs(t, case, dtype)
    mask = {"tree": mask, "shared": mask[0], "chain": None}[kind]
    d_mask = None if mask is None else t.tensor(mask).cuda()
    # what lies behind the drafts never counts, whatever it is
    T = case[0]
    for i, n in enumerate(case[5]):
        k[i, :, n + T:], v[i, :, n + T:] = float("nan"), float("inf")
    out = call("tree_attention", [q, k, v, lengths, d_mask], [t.full_like(q, 7.0)])[0]
    assert status() == 0
    scale = case[3] ** -0.5
    want, size, ulps = O.tree_attention(host(q), host(k), host(v), case[5], mask, scale)
    close(out, want, tree_tolerance(want, size, ulps, dtype))
    again = call("tree_attention", [q, k, v, lengths, d_mask], [t.empty_like(q)])[0]
    assert t.equal(out, again)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("hq", [2, 4, 12, 32])
def test_tree_rows_that_see_nothing_and_masked_poison(t, hq, d, dtype):
    """No committed rows and an empty mask row: zero.  Keys and values of drafts that a row does not see are NaN or
    infinite: they do not reach it."""
    T, hk, cap = 12, 2, 150
    q, k, v, lengths, _ = tree_inputs(t, (T, hq, hk, d, cap, [0, 0, 130]), dtype)
    mask = np.zeros((3, T, T), bool)
    mask[:, np.arange(T), np.arange(T)] = True
    mask[0, 3] = False
    mask[0, 7] = False
    mask[1] = False
    for b, n in ((0, 0), (2, 130)):
        mask[b, :, 5] = False      # nobody sees draft 5
        mask[b, 6, 4] = True       # draft 6 alone sees draft 4 besides itself
        mask[b, 4, 4] = False
        k[b, :, n + 5], v[b, :, n + 5] = float("nan"), float("inf")
        v[b, :, n + 4] = float("inf")
    out = call("tree_attention", [q, k, v, lengths, t.tensor(mask).cuda()], [t.full_like(q, 7.0)])[0]
    kk, vv = host(k), host(v)
    got = host(out)
    assert np.isposinf(got[0, 6]).all() and np.isposinf(got[2, 6]).all()  # a weight times infinity
    vv[:, :, 4 + np.array([0, 130])] = 0  # rows 4 and 134: poison in sequences 0 and 2, clean in 1 (which sees nothing)
    want, size, ulps = O.tree_attention(host(q), np.nan_to_num(kk), np.nan_to_num(vv, posinf=0), [0, 0, 130], mask, d ** -0.5)
    seen = np.ones_like(got, bool)
    seen[[0, 2], 6] = False
    tol = tree_tolerance(want, size, ulps, dtype)
    # sequence 2 reads row 134 only through draft 4, which draft 6 alone sees; committed row 4 of sequence 2 is real
    want2, size2, ulps2 = O.tree_attention(host(q)[2:], np.nan_to_num(kk[2:]), np.nan_to_num(host(v)[2:], posinf=0), [130],
                                           mask[2:], d ** -0.5)
    want[2], tol[2] = want2[0], tree_tolerance(want2, size2, ulps2, dtype)[0]
    assert np.all(np.isfinite(got[seen])) and np.all((np.abs(got - want) <= tol)[seen])
    assert not got[0, 3].any() and not got[0, 7].any() and not got[1].any()
    assert status() == 0


def test_tree_attention_large_scores(t):
    """Scores to +-4000 before the softmax: the running maximum keeps every exponential finite."""
    case = (3, 4, 2, 64, 900, [897, 200])
    for dtype in ("f32", "bf16", "fp16"):
        q, k, v, lengths, mask = tree_inputs(t, case, dtype)
        q, k = q * 30, k * 8
        out = call("tree_attention", [q, k, v, lengths, t.tensor(mask).cuda()], [t.empty_like(q)])[0]
        want, size, ulps = O.tree_attention(host(q), host(k), host(v), case[5], mask, 0.125)
        # 2 e is no longer small: weights change by exp(2 e) - 1, against the largest value in place of the mean
        e = np.expm1(2 * ulps * U) * np.maximum(size, host(v.abs().max()))
        close(out, want, e + (0 if dtype == "f32" else HALF_STEP[dtype]) * size + HALF_STEP[dtype] * np.abs(want) + 1e-7)


def test_tree_attention_scale_and_lengths_that_do_not_fit(t):
    q, k, v, _, mask = tree_inputs(t, (4, 4, 2, 64, 20, [3, 16, 17, 0, 0]), "bf16")
    lengths = [3, 16, 17, -1, 2147483647]
    out = call("tree_attention", [q, k, v, t.tensor(lengths, dtype=t.int32).cuda(), t.tensor(mask).cuda()],
               [t.full_like(q, 7.0)], {"scale": 0.3})[0]
    assert status() == 41 and status() == 0
    want, size, ulps = O.tree_attention(host(q), host(k), host(v), lengths, mask, 0.3)
    close(out, want, tree_tolerance(want, size, ulps, "bf16"))
    assert not out[2:].any()


def test_tree_attention_unaligned(t):
    """Caches and queries one element off alignment."""
    case = (3, 4, 2, 64, 70, [67, 20])
    for dtype in ("bf16", "f32"):
        q, k, v, lengths, mask = tree_inputs(t, case, dtype)
        moved = [values(t, dtype, *x.shape, seed=1, at=1) for x in (q, k, v, q)]
        for m, x in zip(moved, (q, k, v)):
            m.copy_(x)
        out = call("tree_attention", moved[:3] + [lengths, t.tensor(mask).cuda()], [moved[3]])[0]
        want, size, ulps = O.tree_attention(host(q), host(k), host(v), case[5], mask, 0.125)
        close(out, want, tree_tolerance(want, size, ulps, dtype))


def test_tree_attention_past_32_bit_offsets(t):
    """A cache of more than 2**31 elements: the last sequence's rows start past every 32-bit offset."""
    b, hk, cap, d = 3, 16, 350_000, 128
    assert b * hk * cap * d > 1 << 31
    k = t.zeros(b, hk, cap, d, dtype=t.bfloat16, device="cuda")
    v = t.zeros_like(k)
    lengths = [3, 0, 349_000]
    q = values(t, "bf16", b, 2, 32, d, seed=1)
    n = lengths[2]
    k[2, :, n - 500:n + 2] = values(t, "bf16", hk, 502, d, seed=2) * 3
    v[2, :, n - 500:n + 2] = values(t, "bf16", hk, 502, d, seed=3)
    out = call("tree_attention", [q, k, v, t.tensor(lengths, dtype=t.int32).cuda(), None], [t.empty_like(q)])[0]
    # rows of zeros have score 0 and value 0: they only add to the sum
    qq, kk, vv = host(q[2]), host(k[2, :, n - 500:n + 2]), host(v[2, :, n - 500:n + 2])
    for tok in range(2):
        for h in (0, 17, 31):
            s = kk[h // 2, :501 + tok] @ qq[tok, h] * d ** -0.5
            e = np.exp(s)
            total = e.sum() + n - 500
            want = e @ vv[h // 2, :501 + tok] / total
            size = e @ np.abs(vv[h // 2, :501 + tok]) / total
            ulps = (d + 4) * (np.abs(kk[h // 2, :501 + tok]) @ np.abs(qq[tok, h]) * d ** -0.5).max() + n + 16
            got = host(out[2, tok, h])
            assert np.all(np.abs(got - want) <= (2 * ulps * U + 2.0 ** -8) * size + 2.0 ** -8 * np.abs(want) + 1e-7)


# ------------------------------------------------------------------ commit

@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("d,at", [(64, 0), (128, 0), (50, 0), (64, 1), (1, 0)])
def test_commit(t, d, at, dtype):
    b, hk, cap, path_len = 5, 3, 90, 40
    kc, vc = values(t, dtype, b, hk, cap, d, seed=1, at=at), values(t, dtype, b, hk, cap, d, seed=2, at=at)
    k0, v0 = host(kc), host(vc)
    rs = np.random.RandomState(3)
    path = np.sort(np.argsort(rs.rand(b, 50), axis=1)[:, :path_len], axis=1).astype(np.int32)
    path[1] = np.arange(path_len)
    lengths, acc = np.array([0, 7, 40, 11, 89], np.int32), np.array([40, 33, 0, 5, 1], np.int32)
    path[4, 0] = 0
    lengths_d = t.tensor(lengths).cuda()
    outs = call("kv_cache_commit", [lengths_d, t.tensor(path).cuda(), t.tensor(acc).cuda()],
                [kc, vc, t.full((b,), -5, dtype=t.int32, device="cuda")])
    assert status() == 0
    assert np.array_equal(host(kc), O.commit(k0, lengths, path, acc)) and np.array_equal(host(vc), O.commit(v0, lengths, path, acc))
    assert outs[2].tolist() == (lengths + acc).tolist()


def test_commit_refuses_paths_on_the_device(t):
    """Not rising, the same draft twice, negative, outside the cache, too many: rows and length stay."""
    b, cap = 7, 20
    kc, vc = values(t, "bf16", b, 2, cap, 64, seed=1), values(t, "bf16", b, 2, cap, 64, seed=2)
    k0, v0 = kc.clone(), vc.clone()
    path = t.tensor([[2, 1, 3], [1, 1, 2], [-1, 1, 2], [1, 5, 18], [0, 2, 3], [0, 2, 3], [0, 2, 3]], dtype=t.int32).cuda()
    lengths = t.tensor([3, 3, 3, 3, 3, -2, 3], dtype=t.int32).cuda()
    acc = t.tensor([3, 3, 3, 3, 4, 2, 2], dtype=t.int32).cuda()
    outs = call("kv_cache_commit", [lengths, path, acc], [kc, vc, t.zeros_like(lengths)])
    assert status() == 42 and status() == 0
    assert outs[2].tolist() == [3, 3, 3, 3, 3, -2, 5]
    assert t.equal(kc[:6], k0[:6]) and t.equal(vc[:6], v0[:6])
    assert t.equal(kc[6, :, 4], k0[6, :, 5]) and t.equal(vc[6, :, 3], v0[6, :, 3])


# ------------------------------------------------------------------ as they are used

def test_streams_and_graphs(t):
    """On a stream of the caller's, and captured and replayed with other inputs."""
    T, hq, hk, d, cap, b = 4, 8, 2, 64, 500, 3
    steps = t.tensor(rotary.rotary_steps(d)[0]).cuda()
    qw, kw = values(t, "f32", d, seed=1), values(t, "f32", d, seed=2)
    mask = t.tensor(np.tril(np.ones((T, T), bool))).cuda()

    def state(seed, n):
        return dict(qkv=values(t, "bf16", b, T, hq + 2 * hk, d, seed=seed), kc=values(t, "bf16", b, hk, cap, d, seed=seed + 1),
                    vc=values(t, "bf16", b, hk, cap, d, seed=seed + 2), lengths=t.tensor(n, dtype=t.int32).cuda(),
                    pos=t.tensor(n)[:, None].cuda() + t.arange(T).cuda(), q=t.empty(b, T, hq, d, dtype=t.bfloat16, device="cuda"),
                    o=t.empty(b, T, hq, d, dtype=t.bfloat16, device="cuda"))

    def step(s):
        call("qk_norm_rotary_append", [s["qkv"], qw, kw, s["pos"], steps, s["lengths"]], [s["q"], s["kc"], s["vc"]],
             {"num_heads": hq, "kv_num_heads": hk})
        call("tree_attention", [s["q"], s["kc"], s["vc"], s["lengths"], mask], [s["o"]])
        return s["o"]

    first, second = state(30, [0, 100, 496]), state(40, [499 - T, 3, 250])
    want = [step(s).clone() for s in (state(30, [0, 100, 496]), state(40, [499 - T, 3, 250]))]
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        assert t.equal(step(state(30, [0, 100, 496])), want[0])
    t.cuda.current_stream().wait_stream(side)
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g):
        step(first)
    other = t.cuda.CUDAGraph()  # a second graph of the same shapes, replayed in turn
    third = state(40, [499 - T, 3, 250])
    with t.cuda.graph(other):
        step(third)
    for _ in range(2):
        g.replay()
        other.replay()
        assert t.equal(first["o"], want[0]) and t.equal(third["o"], want[1])
    for key in ("qkv", "kc", "vc", "lengths", "pos"):
        first[key].copy_(second[key])
    g.replay()
    assert t.equal(first["o"], want[1])


def test_token_by_token_matches_the_prompt_pass(t):
    """A prompt through qk_norm_rotary and the flash attention, against the same tokens appended and attended one by
    one, in a chunk, and as a tree whose accepted path is committed."""
    B, S, H, D = 2, 128, 4, 64
    qkv = values(t, "bf16", B, S, 3 * H, D, seed=50)
    qw, kw = 1 + 0.1 * values(t, "f32", D, seed=51), 1 + 0.1 * values(t, "f32", D, seed=52)
    steps = t.tensor(rotary.rotary_steps(D)[0]).cuda()
    heads = {"num_heads": H, "kv_num_heads": H}
    packed = call("qk_norm_rotary", [qkv, qw, kw, t.arange(S).cuda(), steps], [t.empty_like(qkv)], heads)[0]
    from hackathon_b200 import _lib as L
    prompt = t.empty(B, S, H * D, dtype=t.bfloat16, device="cuda")
    L.launch(L.K_FLASH_ATTN, [L.make_tensor(packed.data_ptr(), L.BF16, (B, S, 3 * H * D))],
             [L.make_tensor(prompt.data_ptr(), L.BF16, (B, S, H * D))], L.FlashParams(B, S, H, D, D ** -0.5, 1),
             t.cuda.current_stream().cuda_stream)
    prompt = prompt.view(B, S, H, D)
    kc, vc = (t.zeros(B, H, S + 8, D, dtype=t.bfloat16, device="cuda") for _ in range(2))

    def feed(tokens, first, depth, mask):
        n = tokens.shape[1]
        lengths = t.full((B,), first, dtype=t.int32, device="cuda")
        pos = (first + t.tensor(depth)).cuda().expand(B, n).contiguous()
        q = t.empty(B, n, H, D, dtype=t.bfloat16, device="cuda")
        call("qk_norm_rotary_append", [tokens.contiguous(), qw, kw, pos, steps, lengths], [q, kc, vc], heads)
        return call("tree_attention", [q, kc, vc, lengths, mask], [t.empty_like(q)])[0], lengths

    got = [feed(qkv[:, :100], 0, range(100), None)[0]]              # a chunk
    for i in range(100, 120):                                       # token by token
        got.append(feed(qkv[:, i:i + 1], i, [0], None)[0])
    # drafts: tokens 120..127 among wrong ones; the right ones are 0, 2, 3, 5, 6, 8, 9, 10
    right = [0, 2, 3, 5, 6, 8, 9, 10]
    drafts = values(t, "bf16", B, 11, 3 * H, D, seed=53)
    drafts[:, right] = qkv[:, 120:]
    mask, depth = np.zeros((11, 11), bool), np.zeros(11, np.int64)
    for i in range(11):
        before = [j for j in right if j < i]
        mask[i, before] = True
        mask[i, i] = True
        depth[i] = len(before)
    out, lengths = feed(drafts, 120, depth, t.tensor(mask).cuda())
    got.append(out[:, right])
    new = call("kv_cache_commit", [lengths, t.tensor([right] * B, dtype=t.int32).cuda(),
                                   t.tensor([8] * B, dtype=t.int32).cuda()], [kc, vc, t.empty_like(lengths)])[2]
    assert new.tolist() == [S] * B and status() == 0
    # what the cache holds now is the prompt's own keys and values
    assert t.equal(kc[:, :, :S].transpose(1, 2), packed[:, :, H:2 * H]) and t.equal(vc[:, :, :S].transpose(1, 2), packed[:, :, 2 * H:])
    pk = packed.transpose(1, 2)
    want, size, ulps = O.tree_attention(host(packed[:, :, :H]), host(pk[:, H:2 * H]), host(pk[:, 2 * H:]), [0] * B, None, D ** -0.5)
    tol = tree_tolerance(want, size, ulps, "bf16")
    close(t.cat(got, 1), want, tol)
    close(prompt, want, 2 * tol)  # the flash kernel's exponentials have their own 7.5e-5


def test_in_a_native_plan(t):
    """The launches as plan actions on arena offsets, replayed as one CUDA graph."""
    from hackathon_b200 import _lib as L
    from hackathon_b200.kernels import Desc, prepare
    from hackathon_b200.runtime import NativePlan
    B, T, H, D, C = 2, 3, 2, 64, 40
    qkv, kc, vc = values(t, "bf16", B, T, 3 * H, D, seed=1), values(t, "bf16", B, H, C, D, seed=2), values(t, "bf16", B, H, C, D, seed=3)
    steps, lengths, pos = rotary.rotary_steps(D)[0], np.array([5, 37], np.int32), np.array([[5, 6, 7], [37, 38, 39]], np.int64)
    offs, at, host_of = {}, 0, {}
    bits = lambda x: x.view(t.int16).cpu().numpy()  # noqa: E731
    for name, arr in dict(qkv=bits(qkv), kc=bits(kc), vc=bits(vc), steps=steps, lengths=lengths, pos=pos,
                          q=np.zeros((B, T, H, D), np.int16), o=np.zeros((B, T, H, D), np.int16)).items():
        offs[name], host_of[name] = at, np.ascontiguousarray(arr)
        at += (arr.nbytes + 255) // 256 * 256
    plan = NativePlan(at, 1, 0)
    try:
        for name, arr in host_of.items():
            plan.upload(offs[name], arr)
        d = lambda name, dt, *shape: Desc(offs[name], dt, shape, arena=True)  # noqa: E731
        caches = [d("kc", L.BF16, B, H, C, D), d("vc", L.BF16, B, H, C, D)]
        ln = prepare("qk_norm_rotary_append", [d("qkv", L.BF16, B, T, 3 * H, D), None, None, d("pos", L.I64, B, T),
                                               d("steps", L.I64, D // 2), d("lengths", L.I32, B)],
                     [d("q", L.BF16, B, T, H, D)] + caches, {"num_heads": H}).launches
        ln += prepare("tree_attention", [d("q", L.BF16, B, T, H, D)] + caches + [d("lengths", L.I32, B)],
                      [d("o", L.BF16, B, T, H, D)], {}).launches
        for x in ln:
            plan.kernel(0, x)
        plan.finalize(True)
        plan.run()
        got = plan.download(offs["o"], np.zeros((B, T, H, D), np.int16))
    finally:
        plan.close()
    q = t.empty(B, T, H, D, dtype=t.bfloat16, device="cuda")
    d_len = t.tensor(lengths).cuda()
    call("qk_norm_rotary_append", [qkv, None, None, t.tensor(pos).cuda(), t.tensor(steps).cuda(), d_len], [q, kc, vc], {"num_heads": H})
    o = call("tree_attention", [q, kc, vc, d_len], [t.empty_like(q)])[0]
    assert np.array_equal(bits(o), got)


def test_in_a_native_plan_with_a_workspace(t):
    """A cache long enough to be split: the plan's arena holds the workspace; two replays of its graph agree with the
    eager call."""
    from hackathon_b200 import _lib as L
    from hackathon_b200 import kernels as K
    from hackathon_b200.runtime import NativePlan
    B, T, HQ, HK, D, C = 2, 5, 8, 2, 128, 3000
    q, k, v, lengths, mask = tree_inputs(t, (T, HQ, HK, D, C, [2990, 411]), "bf16")
    bits = lambda x: x.view(t.int16).cpu().numpy()  # noqa: E731
    ws = K.tree_attention_workspace(K.Desc(0, L.BF16, (B, T, HQ, D)), K.Desc(0, L.BF16, (B, HK, C, D)))
    assert ws > 0
    host_of = dict(q=bits(q), k=bits(k), v=bits(v), lengths=lengths.cpu().numpy(), mask=mask.astype(np.uint8),
                   o=np.zeros((B, T, HQ, D), np.int16), ws=np.full(ws, 255, np.uint8))
    offs, at = {}, 0
    for name, arr in host_of.items():
        offs[name] = at
        at += (arr.nbytes + 255) // 256 * 256
    plan = NativePlan(at, 1, 0)
    try:
        for name, arr in host_of.items():
            plan.upload(offs[name], np.ascontiguousarray(arr))
        d = lambda name, dt, *shape: K.Desc(offs[name], dt, shape, arena=True)  # noqa: E731
        ln, = K.prepare("tree_attention", [d("q", L.BF16, B, T, HQ, D), d("k", L.BF16, B, HK, C, D), d("v", L.BF16, B, HK, C, D),
                                           d("lengths", L.I32, B), d("mask", L.U8, B, T, T)],
                        [d("o", L.BF16, B, T, HQ, D), d("ws", L.U8, ws)], {}).launches
        plan.kernel(0, ln)
        plan.finalize(True)
        want = bits(call("tree_attention", [q, k, v, lengths, t.tensor(mask).cuda()], [t.empty_like(q)])[0])
        for _ in range(2):
            plan.run()
            assert np.array_equal(plan.download(offs["o"], np.zeros((B, T, HQ, D), np.int16)), want)
    finally:
        plan.close()


def test_general_path_matches_the_native_binding(t):
    """What serves arrays of other libraries, with torch's as the scratch: the same bits."""
    from hackathon_b200 import kernel_registry as R
    q, k, v, lengths, mask = tree_inputs(t, (5, 8, 2, 128, 3000, [2990, 411]), "bf16")
    want = call("tree_attention", [q, k, v, lengths, None], [t.empty_like(q)])[0]
    outs = [t.empty(q.numel(), dtype=q.dtype, device="cuda")]  # flat: comes back in its logical shape
    R._with_workspace(R._make("tree_attention"), "tree_attention", [q, k, v, lengths, None], outs, {})
    t.cuda.synchronize()
    assert len(outs) == 1 and t.equal(outs[0], want)
    outs = call("tree_attention", [q, k, v, lengths, None], [t.empty(q.numel(), dtype=q.dtype, device="cuda")])
    assert outs[0].shape == q.shape and t.equal(outs[0], want)


def test_two_streams_at_once(t):
    """Calls that overlap on the GPU have workspaces of their own."""
    sets = [tree_inputs(t, (9, 16, 2, 128, 20000, [19991, 7000, 13]), "bf16", seed=60 + i) for i in range(2)]
    want = [call("tree_attention", [q, k, v, n, t.tensor(m).cuda()], [t.empty_like(q)])[0] for q, k, v, n, m in sets]
    masks = [t.tensor(s[4]).cuda() for s in sets]
    t.cuda.synchronize()
    streams = [t.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with t.cuda.stream(s):
                q, k, v, n, _ = sets[i]
                got[i].append(call_async("tree_attention", [q, k, v, n, masks[i]], [t.empty_like(q)])[0])
    t.cuda.synchronize()
    for i in range(2):
        assert all(t.equal(x, want[i]) for x in got[i])


def call_async(name, ins, outs, params=None):
    from hackathon_b200.kernel_registry import lookup
    lookup(name)(ins, outs, params or {})
    return outs


@pytest.mark.parametrize("dtype", ["f32", "bf16", "fp16"])
@pytest.mark.parametrize("d,hq", [(64, 2), (64, 12), (128, 4), (128, 40), (96, 24), (256, 2), (17, 2)])
def test_committed_poison_reaches_the_rows_that_see_it(t, d, hq, dtype):
    """A NaN key makes every row of its sequence and kv head NaN; an infinite value makes its dim infinite; another
    sequence and head are as they were."""
    T, hk, cap = 3, 2, 400
    q, k, v, lengths, mask = tree_inputs(t, (T, hq, hk, d, cap, [390, 390, 390]), dtype)
    clean = call("tree_attention", [q, k, v, lengths, t.tensor(mask).cuda()], [t.empty_like(q)])[0]
    k[0, 0, 100] = float("nan")
    v[1, 1, 77, 3] = float("inf")
    out = call("tree_attention", [q, k, v, lengths, t.tensor(mask).cuda()], [t.empty_like(q)])[0]
    g = hq // hk
    assert t.isnan(out[0, :, :g]).all()
    assert t.isposinf(out[1, :, g:, 3]).all()
    keep = t.ones_like(out, dtype=t.bool)
    keep[0, :, :g] = False
    keep[1, :, g:, 3] = False
    assert t.equal(out[keep], clean[keep])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_sequences_and_ragged_lengths(t, dtype):
    """More sequences than a warp has lanes, most of them empty or short, beside one that is long."""
    lengths = [0, 1, 63, 64, 65, 127, 128, 129] * 9 + [2900, 0, 5]
    case = (2, 4, 2, 64, 2999, lengths)
    q, k, v, n, mask = tree_inputs(t, case, dtype)
    out = call("tree_attention", [q, k, v, n, t.tensor(mask).cuda()], [t.full_like(q, 7.0)])[0]
    want, size, ulps = O.tree_attention(host(q), host(k), host(v), lengths, mask, 0.125)
    close(out, want, tree_tolerance(want, size, ulps, dtype))
    assert status() == 0
