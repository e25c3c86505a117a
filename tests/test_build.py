"""The optional torch binding beside the kernel library: what happens where it cannot be built."""

import pytest

from hackathon_b200 import build as B


def test_a_compiler_that_fails_leaves_the_general_path(tmp_path, monkeypatch):
    monkeypatch.setattr(B, "torch_lib", lambda version: tmp_path / "_torch_call.so")
    monkeypatch.setattr(B, "torch_call_command", lambda out: ["sh", "-c", f"echo half > {out}; echo no such header >&2; exit 1"])
    with pytest.warns(UserWarning, match="no such header"):
        B.build_torch_call(force=True)
    assert list(tmp_path.iterdir()) == []


def test_two_builds_write_files_of_their_own(tmp_path, monkeypatch):
    outs = []

    def command(out):
        outs.append(out)
        return ["sh", "-c", f"echo done > {out}"]

    monkeypatch.setattr(B, "torch_lib", lambda version: tmp_path / "_torch_call.so")
    monkeypatch.setattr(B, "torch_call_command", command)
    B.build_torch_call(force=True)
    monkeypatch.setattr(B.os, "getpid", lambda: 1)
    B.build_torch_call(force=True)
    assert outs[0] != outs[1] and [p.name for p in tmp_path.iterdir()] == ["_torch_call.so"]


def test_the_binding_belongs_to_one_torch_and_one_python(tmp_path, monkeypatch):
    """It reads torch's tensors through inlined accessors: another torch's object is not loaded, it is built anew."""
    torch = pytest.importorskip("torch")
    import sysconfig
    from hackathon_b200 import kernel_registry as R
    name = B.torch_lib(str(torch.__version__)).name
    assert str(torch.__version__) in name and sysconfig.get_config_var("SOABI") in name
    assert B.torch_lib("1.0") != B.torch_lib("1.1")
    assert B.torch_version() == str(torch.__version__)
    monkeypatch.setattr(R, "_torch_call", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert R._bound() is False
    monkeypatch.setattr(B, "torch_version", lambda: "0.0.1")
    assert B.torch_call_needs_build()


def test_the_binding_is_used_where_it_is_built(monkeypatch):
    torch = pytest.importorskip("torch")
    from hackathon_b200 import kernel_registry as R
    B.build()
    if not B.torch_lib(str(torch.__version__)).exists():
        pytest.skip("no binding for this torch")
    monkeypatch.setattr(R, "_torch_call", None)
    module = R._bound()
    assert module and module.__file__ == str(B.torch_lib(str(torch.__version__)))
