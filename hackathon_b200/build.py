"""Build ``libc3b200.so`` in-tree with nvcc for sm_100a.

    python -m hackathon_b200.build [--force]

The library is a plain C-ABI shared object (``include/c3b200.h``); Python loads
it with ctypes (``hackathon_b200/_lib.py``).  It links the CUDA runtime
statically and reaches the driver only through cudaGetDriverEntryPoint, so it
loads on any machine with the CUDA driver.
"""

from __future__ import annotations

import argparse
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libc3b200.so"
TORCH_SRC = CSRC / "torch_call.cpp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(CSRC.glob("*.cu"))


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = list(sources()) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return any(p.stat().st_mtime > t for p in deps)


def _torch_dir():
    import importlib.util
    spec = importlib.util.find_spec("torch")
    return Path(spec.origin).parent if spec and spec.origin else None


def torch_version():
    """Version of the torch that is installed, without importing it; None where there is none."""
    torch = _torch_dir()
    if torch is None or not (torch / "version.py").exists():
        return None
    found = re.search(r"^__version__ = ['\"](.+?)['\"]", (torch / "version.py").read_text(), re.M)
    return found.group(1) if found else None


def torch_lib(version) -> Path:
    """The torch binding (fast calls from torch tensors) for one version of torch and this Python.  It reads tensors
    through inlined accessors, so another version's object must not be loaded."""
    return PKG / f"_torch_call.{sysconfig.get_config_var('SOABI')}.torch-{version}.so"


def torch_call_command(out: Path):
    """g++ command of the torch binding, or None where torch or Python's headers are missing."""
    torch, python = _torch_dir(), Path(sysconfig.get_paths()["include"])
    cxx = shutil.which("g++")
    if torch is None or cxx is None or not (python / "Python.h").exists() or not (torch / "lib" / "libc10_cuda.so").exists():
        return None
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    return [cxx, "-O2", "-std=c++20", "-shared", "-fPIC", "-w", str(TORCH_SRC), "-o", str(out), "-I", str(INCLUDE),
            "-I", str(torch / "include"), "-I", str(torch / "include" / "torch" / "csrc" / "api" / "include"),
            "-I", str(python), "-I", str(cuda), "-L", str(torch / "lib"), f"-Wl,-rpath,{torch / 'lib'}",
            "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]


def torch_call_needs_build() -> bool:
    lib = torch_lib(torch_version())
    t = lib.stat().st_mtime if lib.exists() else -1.0
    return any(p.stat().st_mtime > t for p in (TORCH_SRC, INCLUDE / "c3b200.h"))


def build_torch_call(force: bool = False):
    """The binding makes calls from torch tensors faster; without it the registry takes its general path, so a compiler
    that fails on torch's headers is a warning."""
    if not force and not torch_call_needs_build():
        return
    lib = torch_lib(torch_version())
    tmp = lib.with_suffix(f".{os.getpid()}.tmp")
    cmd = torch_call_command(tmp)
    if cmd is None:
        return
    done = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if done.returncode == 0:
        os.replace(tmp, lib)
        return
    tmp.unlink(missing_ok=True)
    warnings.warn("the torch binding was not built: " + done.stdout.decode(errors="replace")[-2000:])


def build(force: bool = False, verbose: bool = False) -> Path:
    build_torch_call(force)
    if not force and not needs_build():
        return LIB
    objdir = ROOT / "_build"
    objdir.mkdir(exist_ok=True)
    objs = []
    common = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-I", str(INCLUDE), "-I", str(CSRC), "--expt-relaxed-constexpr", "-rdc=true"]
    if verbose:
        common += ["-Xptxas", "-v"]
    procs = []
    for src in sources():
        obj = objdir / (src.stem + ".o")
        objs.append(obj)
        cmd = common + ["-c", str(src), "-o", str(obj)]
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for cmd, pr in procs:
        out, _ = pr.communicate()
        if pr.returncode != 0 or verbose:
            sys.stderr.write(out.decode(errors="replace"))
        if pr.returncode != 0:
            raise RuntimeError("nvcc failed: " + " ".join(cmd))
    tmp = LIB.with_suffix(".so.tmp")
    link = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
    subprocess.run(link, check=True)
    os.replace(tmp, LIB)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))


if __name__ == "__main__":
    main()
