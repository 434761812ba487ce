# SPDX-License-Identifier: Apache-2.0
"""Build of the sm_100a shared library `libqdq_b200.so` (C ABI in include/qdq_b200.h)
and of `libqdq_b200_torch.so`, the torch.library kernels that call it.

The first is compiled in-tree with nvcc (no torch headers, no JIT cache), the
second, csrc/torch_ops.cpp, with the host compiler against the installed
torch; both sit next to this package and travel with the source tree.  They go
stale apart: the second also where another torch is installed than the one it
was compiled against.  What needs the C ABI alone does not need the second.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import tempfile
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
PLUGIN_ROOT = PKG_DIR.parent                       # vllm-qdq-plugin_b200/
CSRC_DIR = PLUGIN_ROOT / "csrc"
INCLUDE_DIR = PLUGIN_ROOT.parent / "include"       # repo-level public header
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libqdq_b200.so"
TORCH_OPS_SOURCE = CSRC_DIR / "torch_ops.cpp"
TORCH_OPS_PATH = LIB_DIR / "libqdq_b200_torch.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
# No --use_fast_math / -ftz: bf16/fp32 subnormals must survive for bit-exact QDQ.
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-shared",
              "--expt-relaxed-constexpr"]


def sources() -> list[Path]:
    return sorted(CSRC_DIR.glob("*.cu"))


def _newer(built: Path, inputs: list[Path]) -> bool:
    return not built.exists() or any(p.stat().st_mtime > built.stat().st_mtime for p in inputs)


def is_stale() -> bool:
    return _newer(LIB_PATH, sources() + sorted(CSRC_DIR.glob("*.cuh")) + sorted(INCLUDE_DIR.glob("*.h")))


def _built_for() -> str:
    """What libqdq_b200_torch.so is tied to; it carries this text."""
    import torch

    return f"qdq torch ops for torch {torch.__version__} cuda {torch.version.cuda} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)};"


def ops_are_stale() -> bool:
    return (_newer(TORCH_OPS_PATH, [TORCH_OPS_SOURCE] + sorted(INCLUDE_DIR.glob("*.h")))
            or _built_for().encode() not in TORCH_OPS_PATH.read_bytes())


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: cannot build libqdq_b200.so for sm_100a")


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")


def _has_nostdlibxx(cxx: str) -> bool:
    """Whether the compiler knows -nostdlib++ (GCC from 13 on)."""
    with tempfile.TemporaryDirectory() as tmp:
        cmd = [cxx, "-shared", "-nostdlib++", "-x", "c++", os.devnull, "-o", f"{tmp}/empty.so"]
        return subprocess.run(cmd, capture_output=True).returncode == 0


def _torch_ops_commands(obj: Path, out: Path) -> tuple[list[str], list[str]]:
    """Compile and link commands of the torch.library kernels."""
    import torch
    from torch.utils import cpp_extension

    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        raise RuntimeError("g++ not found: cannot build libqdq_b200_torch.so")
    cuda = Path(nvcc_path()).resolve().parent.parent
    includes = [f"-I{INCLUDE_DIR}", *(f"-isystem{p}" for p in cpp_extension.include_paths()), f"-isystem{cuda / 'include'}"]
    compile_cmd = [cxx, "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                   f'-DQDQ_BUILT_FOR="{_built_for()}"', *includes, "-c", "-o", str(obj), str(TORCH_OPS_SOURCE)]
    # The shared libstdc++ by name: a toolchain that links a static one in would give this library its own exception
    # machinery, and an error it raises would end the process instead of reaching Python.
    link_cmd = [cxx, "-shared", *(["-nostdlib++"] if _has_nostdlibxx(cxx) else []), "-o", str(out), str(obj), "-l:libstdc++.so.6",
                f"-L{LIB_DIR}", "-lqdq_b200", *(f"-L{p}" for p in cpp_extension.library_paths()), "-lc10", "-lc10_cuda",
                "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-Wl,-rpath,$ORIGIN"]
    return compile_cmd, link_cmd


class _TorchOps:
    """One build of libqdq_b200_torch.so: compiled beside the C ABI library, linked against it."""

    def __init__(self, obj_dir: Path, verbose: bool):
        self._obj, self._verbose = obj_dir / "torch_ops.o", verbose
        self._tmp = TORCH_OPS_PATH.with_name(f".{TORCH_OPS_PATH.name}.{os.getpid()}.tmp")

    def compile(self) -> None:
        cmd, self._link = _torch_ops_commands(self._obj, self._tmp)
        _run(cmd, self._verbose)

    def link(self) -> None:
        _run(self._link, self._verbose)
        os.replace(self._tmp, TORCH_OPS_PATH)


def build_ops(force: bool = False, verbose: bool = False) -> Path:
    """Build libqdq_b200_torch.so where it is missing or stale (the C ABI library first)."""
    build_native(verbose=verbose)
    if force or ops_are_stale():
        with tempfile.TemporaryDirectory() as tmp:
            ops = _TorchOps(Path(tmp), verbose)
            ops.compile()
            ops.link()
    return TORCH_OPS_PATH


def build_native(force: bool = False, verbose: bool = False) -> Path:
    """Compile every csrc/*.cu into one sm_100a shared library (idempotent), and csrc/torch_ops.cpp with them where its
    own library is stale; that one may fail here (`build_ops`, which needs it, then raises).

    Each translation unit is compiled to an object file in parallel (one compiler
    per source), then the objects are linked into the shared libraries."""
    if not force and not is_stale():
        return LIB_PATH
    from concurrent.futures import ThreadPoolExecutor

    LIB_DIR.mkdir(parents=True, exist_ok=True)
    obj_dir = LIB_DIR / f".obj.{os.getpid()}"
    obj_dir.mkdir(exist_ok=True)
    compile_flags = [f for f in NVCC_FLAGS if f != "-shared"]
    jobs = []
    for src in sources():
        obj = obj_dir / (src.stem + ".o")
        jobs.append((obj, [nvcc_path(), *ARCH_FLAGS, *compile_flags, f"-I{INCLUDE_DIR}", f"-I{CSRC_DIR}",
                           "-c", "-o", str(obj), str(src)]))
    ops = _TorchOps(obj_dir, verbose)

    def compile_ops() -> bool:
        if not force and not ops_are_stale():
            return False
        ops.compile()
        return True

    try:
        with ThreadPoolExecutor(max_workers=max(1, min(len(jobs) + 1, os.cpu_count() or 1))) as pool:
            ops_done = pool.submit(compile_ops)
            for fut in [pool.submit(_run, cmd, verbose) for _, cmd in jobs]:
                fut.result()
        tmp = LIB_PATH.with_name(f".{LIB_PATH.name}.{os.getpid()}.tmp")
        _run([nvcc_path(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", str(tmp),
              *[str(o) for o, _ in jobs]], verbose)
        os.replace(tmp, LIB_PATH)
        try:
            if ops_done.result():
                ops.link()
        except Exception as e:  # no torch, its headers or a host compiler: the C ABI needs none of them
            from ._log import init_logger
            init_logger(__name__).warning("libqdq_b200_torch.so was not built, the MXFP8 operators cannot be called: %s", e)
    finally:
        shutil.rmtree(obj_dir, ignore_errors=True)
    return LIB_PATH
