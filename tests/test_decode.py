"""Cached decoding without a GPU: phase steps, the names, and every refusal, which comes before any CUDA call."""

import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

from hackathon_b200 import _lib as L
from hackathon_b200 import kernels as K
from hackathon_b200 import rotary
from hackathon_b200.kernels import Desc

NAMES = {"rotary_embedding": L.K_ROTARY, "qk_norm_rotary": L.K_QK_NORM_ROTARY,
         "qk_norm_rotary_append": L.K_QK_NORM_APPEND, "tree_attention": L.K_TREE_ATTN,
         "kv_cache_commit": L.K_KV_COMMIT}


def test_names_resolve_in_both_registries():
    from hackathon_b200 import kernel_registry as R
    for name, kid in NAMES.items():
        assert L.kernel_id(name) == kid
        assert R.is_registered(name)


def test_phase_steps_are_turns():
    f = rotary.rotary_frequencies(8, 10000.0)
    assert np.allclose(f, [1.0, 0.1, 0.01, 0.001])
    steps = rotary.phase_steps(f)
    assert steps.dtype == np.int64
    # one position adds f / 2 pi turns, to the precision of the float64 frequency
    assert np.allclose(steps.astype(np.float64) / 2.0 ** 64 * 2 * math.pi, f, rtol=1e-15)
    # a whole turn more is the same step; a backward turn is the complement
    assert rotary.phase_steps([-1.0])[0] == -steps[0]


@pytest.mark.parametrize("pos", [1, 4095, 131071, (1 << 31) - 1])
def test_far_positions_keep_their_angle(pos):
    """The wrapped product against exact integer arithmetic: range reduction adds nothing to the
    step's own rounding (2**-53 of a frequency)."""
    f = rotary.rotary_frequencies(64, 500000.0)
    steps = rotary.phase_steps(f)
    with np.errstate(over="ignore"):
        phase = np.uint64(pos) * steps.view(np.uint64)
    for i in (0, 7, 31):
        exact = pos * int(math.ldexp(f[i] / (2 * math.pi), 64)) % 2 ** 64
        assert int(phase[i]) == exact


def test_scalings():
    plain, one = rotary.rotary_steps(64)
    assert one == 1.0
    linear, one = rotary.rotary_steps(64, scaling="linear", factor=4.0)
    assert one == 1.0 and np.all(np.abs(linear * 4 - plain) <= 4)
    base, one = rotary.rotary_steps(64, scaling="base", factor=8.0)
    assert one == 1.0 and base[0] == plain[0]
    assert abs(base[-1] / plain[-1] - 1 / 8.0) < 1e-12
    turns, scale = rotary.rotary_steps(64, scaling="turns", factor=32.0, original_length=4096)
    assert scale == pytest.approx(0.1 * math.log(32.0) + 1.0)
    assert turns[0] == plain[0]                                  # 650 turns in 4096 positions: as trained
    assert abs(turns[-1] / plain[-1] - 1 / 32.0) < 1e-12         # less than one turn: slowed whole
    assert np.all(np.diff(turns) < 0)


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0),
                                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="other"),
                                dict(rotary_dim=2, scaling="base", factor=2.0),
                                dict(rotary_dim=8, scaling="turns", beta_fast=1.0, beta_slow=1.0)])
def test_rotary_steps_refuses(kw):
    with pytest.raises(ValueError):
        rotary.rotary_steps(**kw)


def test_phase_steps_refuses_what_is_not_finite():
    with pytest.raises(ValueError):
        rotary.phase_steps([1.0, float("inf")])


def test_parameter_blocks_match_the_header(tmp_path):
    structs = {"c3b_rotary_params": L.RotaryParams, "c3b_qk_norm_params": L.QkNormParams,
               "c3b_tree_attn_params": L.TreeAttnParams, "c3b_kv_commit_params": L.KvCommitParams}
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "c3b200.h"\nint main(void){\n'
    for name, cls in structs.items():
        src += f'printf("{name} %zu\\n", sizeof({name}));\n'
        for field, _ in cls._fields_:
            src += f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));\n'
    (tmp_path / "s.c").write_text(src + "return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls), name
        for field, _ in cls._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(cls, field).offset, f"{name}.{field}"


class Space:
    """Made-up addresses that are never dereferenced, 1 MiB apart."""

    def __init__(self):
        self.at = 1 << 20

    def __call__(self, dtype, *shape):
        self.at += 1 << 20
        return Desc(self.at, dtype, tuple(shape))


def launch(name, ins, outs, params):
    prep = K.prepare(name, ins, outs, params)
    for ln in prep.launches:
        L.launch(ln.kid, ln.ins, ln.outs, ln.params)


B, S, HQ, HK, D, C = 2, 3, 4, 2, 64, 16
HEADS = {"num_heads": HQ, "kv_num_heads": HK}


def rotary_call(**k):
    n = Space()
    a = dict(x=n(L.BF16, B, S, HQ, D), pos=n(L.I64, B, S), steps=n(L.I64, D // 2), out=n(L.BF16, B, S, HQ, D))
    a.update({key: v(n) if callable(v) else v for key, v in k.items()})
    return "rotary_embedding", [a["x"], a["pos"], a["steps"]], [a["out"]], {}


def norm_call(params=None, **k):
    n = Space()
    w = HQ + 2 * HK
    a = dict(x=n(L.F16, B, S, w, D), qw=n(L.F32, D), kw=n(L.F32, HK, D), pos=n(L.I32, S), steps=n(L.I64, D // 4),
             out=n(L.F16, B, S, w, D))
    a.update({key: v(n) if callable(v) else v for key, v in k.items()})
    return "qk_norm_rotary", [a[i] for i in ("x", "qw", "kw", "pos", "steps")], [a["out"]], {**HEADS, **(params or {})}


def append_call(params=None, **k):
    n = Space()
    a = dict(x=n(L.F32, B, S, (HQ + 2 * HK) * D), qw=None, kw=None, pos=n(L.I32, B, S), steps=n(L.I64, 8),
             lengths=n(L.I32, B), q=n(L.F32, B, S, HQ, D), k=n(L.F32, B, HK, C, D), v=n(L.F32, B, HK, C, D))
    a.update({key: v(n) if callable(v) else v for key, v in k.items()})
    return ("qk_norm_rotary_append", [a[i] for i in ("x", "qw", "kw", "pos", "steps", "lengths")],
            [a["q"], a["k"], a["v"]], {**HEADS, **(params or {})})


def tree_call(params=None, **k):
    n = Space()
    a = dict(q=n(L.BF16, B, S, HQ, D), k=n(L.BF16, B, HK, C, D), v=n(L.BF16, B, HK, C, D), lengths=n(L.I32, B),
             mask=n(L.U8, B, S, S), out=n(L.BF16, B, S, HQ, D))
    a.update({key: v(n) if callable(v) else v for key, v in k.items()})
    return "tree_attention", [a[i] for i in ("q", "k", "v", "lengths", "mask")], [a["out"]], params or {}


def commit_call(**k):
    n = Space()
    a = dict(lengths=n(L.I32, B), path=n(L.I32, B, 3), acc=n(L.I32, B), k=n(L.F16, B, HK, C, D),
             v=n(L.F16, B, HK, C, D), new=n(L.I32, B))
    a.update({key: v(n) if callable(v) else v for key, v in k.items()})
    return "kv_cache_commit", [a["lengths"], a["path"], a["acc"]], [a["k"], a["v"], a["new"]], {}


REFUSED = {
    "rotary: output of another type": rotary_call(out=lambda n: n(L.F32, B, S, HQ, D)),
    "rotary: output of another size": rotary_call(out=lambda n: n(L.BF16, B, S, HQ, D + 8)),
    "rotary: whole numbers": rotary_call(x=lambda n: n(L.I32, B, S, HQ, D), out=lambda n: n(L.I32, B, S, HQ, D)),
    "rotary: rank": rotary_call(x=lambda n: n(L.BF16, B * S, HQ, D)),
    "rotary: float positions": rotary_call(pos=lambda n: n(L.F32, B, S)),
    "rotary: positions of another batch": rotary_call(pos=lambda n: n(L.I64, B + 1, S)),
    "rotary: more pairs than the head has": rotary_call(steps=lambda n: n(L.I64, D // 2 + 1)),
    "rotary: no pairs": rotary_call(steps=lambda n: n(L.I64, 0)),
    "rotary: steps as floats": rotary_call(steps=lambda n: n(L.F32, D // 2)),
    "rotary: output half over the input": rotary_call(x=Desc(1 << 20, L.BF16, (B, S, HQ, D)),
                                                      out=Desc((1 << 20) + 128, L.BF16, (B, S, HQ, D))),
    "rotary: output over the positions": rotary_call(pos=Desc(1 << 30, L.I64, (B, S)), out=Desc(1 << 30, L.BF16, (B, S, HQ, D))),
    "rotary: a token of more than 2**31 elements": rotary_call(x=lambda n: n(L.BF16, 1, 1, 1 << 23, 256), pos=lambda n: n(L.I64, 1, 1),
                                                               out=lambda n: n(L.BF16, 1, 1, 1 << 23, 256)),
    "norm: output over a weight": norm_call(qw=Desc(1 << 30, L.F32, (D,)), out=Desc(1 << 30, L.F16, (B, S, HQ + 2 * HK, D))),
    "append: cache over the lengths": append_call(lengths=Desc(1 << 30, L.I32, (B,)), k=Desc(1 << 30, L.F32, (B, HK, C, D))),
    "norm: heads do not add up": norm_call({"kv_num_heads": 1}),
    "norm: weights without normalisation": norm_call({"normalize": 0}),
    "norm: weight of another size": norm_call(qw=lambda n: n(L.F32, D // 2)),
    "norm: 16-bit weight": norm_call(kw=lambda n: n(L.F16, HK, D)),
    "norm: negative heads": norm_call({"num_heads": -4, "kv_num_heads": 6}),
    "norm: width not a multiple of the heads": norm_call(x=lambda n: n(L.F16, B, S, (HQ + 2 * HK) * D + 1)),
    "append: caches of different capacity": append_call(v=lambda n: n(L.F32, B, HK, C + 1, D)),
    "append: caches of another batch": append_call(k=lambda n: n(L.F32, B + 1, HK, C, D),
                                                   v=lambda n: n(L.F32, B + 1, HK, C, D)),
    "append: caches of another type": append_call(k=lambda n: n(L.F16, B, HK, C, D)),
    "append: lengths int64": append_call(lengths=lambda n: n(L.I64, B)),
    "append: q of another size": append_call(q=lambda n: n(L.F32, B, S, HQ + 1, D)),
    "append: one buffer for both caches": append_call(k=Desc(1 << 30, L.F32, (B, HK, C, D)),
                                                      v=Desc(1 << 30, L.F32, (B, HK, C, D))),
    "tree: caches of another head size": tree_call(k=lambda n: n(L.BF16, B, HK, C, 32),
                                                   v=lambda n: n(L.BF16, B, HK, C, 32)),
    "tree: heads not a multiple": tree_call(k=lambda n: n(L.BF16, B, 3, C, D), v=lambda n: n(L.BF16, B, 3, C, D)),
    "tree: mixed types": tree_call(v=lambda n: n(L.F16, B, HK, C, D)),
    "tree: mask of another size": tree_call(mask=lambda n: n(L.U8, B, S, S + 1)),
    "tree: mask as floats": tree_call(mask=lambda n: n(L.F32, B, S, S)),
    "tree: lengths int64": tree_call(lengths=lambda n: n(L.I64, B)),
    "tree: head size": tree_call(q=lambda n: n(L.BF16, B, S, HQ, 264), out=lambda n: n(L.BF16, B, S, HQ, 264),
                                 k=lambda n: n(L.BF16, B, HK, C, 264), v=lambda n: n(L.BF16, B, HK, C, 264)),
    "tree: output over q": tree_call(q=Desc(1 << 30, L.BF16, (B, S, HQ, D)), out=Desc(1 << 30, L.BF16, (B, S, HQ, D))),
    "tree: output of another type": tree_call(out=lambda n: n(L.F32, B, S, HQ, D)),
    "tree: scale is no number": tree_call({"scale": float("nan")}),
    "tree: negative scale": tree_call({"scale": -0.125}),
    "tree: scale that overflows in powers of two": tree_call({"scale": 3e38}),
    "tree: no workspace": tree_call(k=lambda n: n(L.BF16, B, HK, 600, D), v=lambda n: n(L.BF16, B, HK, 600, D)),
    "tree: workspace too small": (lambda c: (c[0], c[1], c[2] + [Desc(1 << 30, L.U8, (1000,))], c[3]))(
        tree_call(k=lambda n: n(L.BF16, B, HK, 600, D), v=lambda n: n(L.BF16, B, HK, 600, D))),
    "commit: path int64": commit_call(path=lambda n: n(L.I64, B, 3)),
    "commit: path rank": commit_call(path=lambda n: n(L.I32, B)),
    "commit: accepted of another size": commit_call(acc=lambda n: n(L.I32, B + 1)),
    "commit: new lengths over lengths": commit_call(lengths=Desc(1 << 30, L.I32, (B,)), new=Desc(1 << 30, L.I32, (B,))),
    "commit: caches differ": commit_call(v=lambda n: n(L.F16, B, HK, C + 1, D)),
    "commit: whole-number caches": commit_call(k=lambda n: n(L.I32, B, HK, C, D), v=lambda n: n(L.I32, B, HK, C, D)),
}


@pytest.mark.parametrize("case", sorted(REFUSED))
def test_refused_without_gpu_work(case):
    with pytest.raises((ValueError, RuntimeError), match=r"^(?!.*(CUDA|cuTensorMap))"):  # not a launch that only the missing GPU stopped
        launch(*REFUSED[case])


@pytest.mark.parametrize("call", [
    rotary_call(x=lambda n: n(L.BF16, 0, S, HQ, D), out=lambda n: n(L.BF16, 0, S, HQ, D), pos=lambda n: n(L.I64, 0, S)),
    rotary_call(x=lambda n: n(L.BF16, B, 0, HQ, D), out=lambda n: n(L.BF16, B, 0, HQ, D), pos=lambda n: n(L.I64, B, 0)),
    tree_call(q=lambda n: n(L.BF16, B, 0, HQ, D), out=lambda n: n(L.BF16, B, 0, HQ, D), mask=None),
])
def test_empty_calls_launch_nothing(call):
    launch(*call)
