# SPDX-License-Identifier: Apache-2.0
"""Build of the sm_100a shared library `libqdq_b200.so` (C ABI in include/qdq_b200.h)
and of `libqdq_b200_torch.so`, the torch.library kernels that call it.

The first is compiled in-tree with nvcc (no torch headers, no JIT cache), the
second, csrc/torch_ops.cpp, with the host compiler against the installed
torch; both sit next to this package and travel with the source tree.
"""

from __future__ import annotations

import os
import shutil
import subprocess
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


def _inputs() -> list[Path]:
    return sources() + [TORCH_OPS_SOURCE] + sorted(CSRC_DIR.glob("*.cuh")) + sorted(INCLUDE_DIR.glob("*.h"))


def is_stale() -> bool:
    if not LIB_PATH.exists() or not TORCH_OPS_PATH.exists():
        return True
    built = min(LIB_PATH.stat().st_mtime, TORCH_OPS_PATH.stat().st_mtime)
    return any(p.stat().st_mtime > built for p in _inputs())


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
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")


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
                   *includes, "-c", "-o", str(obj), str(TORCH_OPS_SOURCE)]
    # The shared libstdc++ by name: a toolchain that links a static one in would give this library its own exception
    # machinery, and an error it raises would end the process instead of reaching Python.
    link_cmd = [cxx, "-shared", "-nostdlib++", "-o", str(out), str(obj), "-l:libstdc++.so.6", f"-L{LIB_DIR}", "-lqdq_b200",
                *(f"-L{p}" for p in cpp_extension.library_paths()), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
                "-Wl,-rpath,$ORIGIN"]
    return compile_cmd, link_cmd


def build_native(force: bool = False, verbose: bool = False) -> Path:
    """Compile every csrc/*.cu into one sm_100a shared library, and csrc/torch_ops.cpp
    into the one that registers the torch.library kernels (idempotent).

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
    ops_obj = obj_dir / "torch_ops.o"
    ops_tmp = TORCH_OPS_PATH.with_name(f".{TORCH_OPS_PATH.name}.{os.getpid()}.tmp")
    ops_compile, ops_link = _torch_ops_commands(ops_obj, ops_tmp)
    try:
        with ThreadPoolExecutor(max_workers=max(1, min(len(jobs) + 1, os.cpu_count() or 1))) as pool:
            for fut in [pool.submit(_run, cmd, verbose) for cmd in [ops_compile, *(c for _, c in jobs)]]:
                fut.result()
        tmp = LIB_PATH.with_name(f".{LIB_PATH.name}.{os.getpid()}.tmp")
        _run([nvcc_path(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", str(tmp),
              *[str(o) for o, _ in jobs]], verbose)
        os.replace(tmp, LIB_PATH)
        _run(ops_link, verbose)
        os.replace(ops_tmp, TORCH_OPS_PATH)
    finally:
        shutil.rmtree(obj_dir, ignore_errors=True)
    return LIB_PATH
