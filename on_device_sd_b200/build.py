"""Builds libb200moe.so in-tree with nvcc for sm_100a (no other architecture is supported), and _step.so, the
tensor entry points of the step operators (csrc/bindings.cpp), with the host compiler against the installed torch.

    python -m on_device_sd_b200.build [--force] [--verbose] [--lib-only]

--lib-only leaves _step.so out: C callers of libb200moe.so need neither torch's nor Python's headers.

The shared libraries land next to this file so that they travel with the source tree; nothing
is installed into site-packages and no JIT cache is used.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB = PKG / "libb200moe.so"
STEP = PKG / "_step.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr", "--extended-lambda",
]


def _defines() -> list[str]:
    d = []
    if (CSRC / "ffn_int4.cuh").exists():
        d.append("-DB200MOE_WITH_INT4")
    if (CSRC / "ffn_umma.cuh").exists():
        d.append("-DB200MOE_WITH_UMMA")
    return d


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + [CSRC / "internal.h", PKG.parent / "include" / "b200moe.h", Path(__file__)]
    return any(p.stat().st_mtime > t for p in deps)


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; libb200moe.so cannot be built")


def step_tag() -> str:
    """What _step.so has to be compiled against to be loaded here: it uses torch's C++ interface and Python's."""
    import sysconfig

    import torch
    return f"torch {torch.__version__} cxx11abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} {sysconfig.get_config_var('SOABI')}"


def built_for(path: Path) -> str | None:
    """The step_tag that a _step.so was built with, without loading it (with other libraries that may not even fail cleanly)."""
    m = re.search(rb"b200moe_step built for <([^>\0]*)>", path.read_bytes())
    return m.group(1).decode() if m else None


def _step_is_current() -> bool:
    deps = (CSRC / "bindings.cpp", CSRC / "overlap.h", PKG.parent / "include" / "b200moe.h", Path(__file__))
    return STEP.exists() and all(p.stat().st_mtime <= STEP.stat().st_mtime for p in deps) and built_for(STEP) == step_tag()


def _build_step(force: bool, verbose: bool) -> None:
    if not force and _step_is_current():
        return
    import sysconfig

    import torch
    src = CSRC / "bindings.cpp"
    tdir = Path(torch.__file__).parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    cxx = os.environ.get("CXX") or shutil.which("g++") or "g++"
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DB200MOE_STEP_TAG="{step_tag()}"', "-isystem", sysconfig.get_paths()["include"], "-isystem", str(tdir / "include"), "-isystem", str(cuda / "include"),
           str(src), "-o", str(STEP), "-L", str(tdir / "lib"), "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lc10_cuda", "-ltorch_cuda",
           "-L", str(PKG), "-lb200moe", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError("the host compiler failed building _step.so:\n" + res.stderr[-4000:])


def build(force: bool = False, verbose: bool = False, step: bool = True) -> Path:
    if not force and not _stale():
        if step:
            _build_step(False, verbose)
        return LIB
    import tempfile
    from concurrent.futures import ThreadPoolExecutor
    nvcc = nvcc_path()
    flags = [*NVCC_FLAGS, *_defines(), "-I", str(PKG.parent / "include"), *(["-Xptxas", "-v"] if verbose else [])]
    with tempfile.TemporaryDirectory() as tmp:
        def compile_one(src: Path):
            obj = Path(tmp) / (src.stem + ".o")
            return obj, subprocess.run([nvcc, *flags, "-c", str(src), "-o", str(obj)], capture_output=True, text=True)

        with ThreadPoolExecutor() as pool:
            done = list(pool.map(compile_one, _sources()))
        for _, res in done:
            if verbose or res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError("nvcc failed building libb200moe.so:\n" + res.stderr[-4000:])
        cmd = [nvcc, *NVCC_FLAGS, "-shared", "-o", str(LIB), *[str(o) for o, _ in done]]
        cmd += ["-lcuda"] if (CSRC / "ffn_umma.cuh").exists() else []
        res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed building libb200moe.so:\n" + res.stderr[-4000:])
    if step:
        _build_step(True, verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, step="--lib-only" not in sys.argv)
    print(LIB)
