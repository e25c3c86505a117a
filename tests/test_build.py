"""The optional torch binding beside the kernel library: what happens where it cannot be built."""

import pytest

from hackathon_b200 import build as B


def test_a_compiler_that_fails_leaves_the_general_path(tmp_path, monkeypatch):
    monkeypatch.setattr(B, "TORCH_LIB", tmp_path / "_torch_call.so")
    monkeypatch.setattr(B, "torch_call_command", lambda out: ["sh", "-c", f"echo half > {out}; echo no such header >&2; exit 1"])
    with pytest.warns(UserWarning, match="no such header"):
        B.build_torch_call(force=True)
    assert list(tmp_path.iterdir()) == []


def test_two_builds_write_files_of_their_own(tmp_path, monkeypatch):
    outs = []

    def command(out):
        outs.append(out)
        return ["sh", "-c", f"echo done > {out}"]

    monkeypatch.setattr(B, "TORCH_LIB", tmp_path / "_torch_call.so")
    monkeypatch.setattr(B, "torch_call_command", command)
    B.build_torch_call(force=True)
    monkeypatch.setattr(B.os, "getpid", lambda: 1)
    B.build_torch_call(force=True)
    assert outs[0] != outs[1] and [p.name for p in tmp_path.iterdir()] == ["_torch_call.so"]
