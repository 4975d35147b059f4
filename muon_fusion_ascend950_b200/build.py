"""In-tree build of the two native libraries of this package.

* ``libmuon_polar_sm100.so`` -- the sm_100a kernels and the C ABI declared in
  ``include/muon_polar_sm100.h`` (nvcc, static CUDA runtime, no torch): the
  Polar Express step (``muon_polar_sm100.cu``), the Muon update around it
  (``muon_update_sm100.cu``) and the training-step operators declared in
  ``include/muon_train_sm100.h`` (``distill_topk_sm100.cu``,
  ``residual_norm_sm100.cu``, ``route_experts_sm100.cu``, ``attention_sm100.cu``,
  ``rotary_sm100.cu``, ``clip_grads_sm100.cu``).
* ``_C.so`` -- the PyTorch operators ``muon_ascend950::*`` on the CUDA
  dispatch key (``polar_step_op.cpp``, ``train_ops.cpp``, ``block_ops.cpp``,
  and ``clip_list.cpp`` beside them), linked against the library above (rpath ``$ORIGIN``).

Both land next to this file so that they travel with the source tree.  Each
source compiles to an object under ``_build/`` (all in parallel); what is newer
than every input is not built again, a library without its objects included.  Run with
``python -m muon_fusion_ascend950_b200.build`` (``--force`` to rebuild).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
REPO = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = REPO / "include"
BUILD = PKG / "_build"
LIB_NAME = "libmuon_polar_sm100.so"
OP_NAME = "_C.so"

NVCC_ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _cuda_home() -> Path:
    home = os.environ.get("CUDA_HOME") or os.environ.get("CUDA_PATH")
    if home:
        return Path(home)
    nvcc = shutil.which("nvcc")
    if nvcc:
        return Path(nvcc).resolve().parent.parent
    return Path("/usr/local/cuda")


def _newer(target: Path, sources) -> bool:
    if not target.exists():
        return False
    t = target.stat().st_mtime
    return all(Path(s).stat().st_mtime <= t for s in sources)


def _run(cmd) -> None:
    print("+", " ".join(str(c) for c in cmd), flush=True)
    subprocess.run([str(c) for c in cmd], check=True, cwd=REPO)


CU_SOURCES = {  # source -> the headers it includes
    "muon_polar_sm100.cu": ["sm100_ptx.cuh", "muon_polar_sm100.h"],
    "muon_update_sm100.cu": ["sm100_ptx.cuh", "muon_polar_sm100.h"],
    "distill_topk_sm100.cu": ["train_common.cuh", "sm100_ptx.cuh", "muon_train_sm100.h", "muon_polar_sm100.h"],
    "residual_norm_sm100.cu": ["train_common.cuh", "sm100_ptx.cuh", "muon_train_sm100.h", "muon_polar_sm100.h"],
    "route_experts_sm100.cu": ["train_common.cuh", "sm100_ptx.cuh", "muon_train_sm100.h", "muon_polar_sm100.h"],
    "attention_sm100.cu": ["tcgen05_attention.cuh", "train_common.cuh", "sm100_ptx.cuh", "muon_train_sm100.h", "muon_polar_sm100.h"],
    "rotary_sm100.cu": ["train_common.cuh", "sm100_ptx.cuh", "muon_train_sm100.h", "muon_polar_sm100.h"],
    "clip_grads_sm100.cu": ["train_common.cuh", "sm100_ptx.cuh", "muon_train_sm100.h", "muon_polar_sm100.h"],
}
OP_SOURCES = {
    "polar_step_op.cpp": ["muon_polar_sm100.h"],
    "train_ops.cpp": ["train_ops_common.h", "muon_train_sm100.h", "muon_polar_sm100.h"],
    "block_ops.cpp": ["train_ops_common.h", "muon_train_sm100.h", "muon_polar_sm100.h"],
    "clip_list.cpp": ["train_ops_common.h", "muon_train_sm100.h", "muon_polar_sm100.h"],
}


def _inputs(name: str, headers) -> list:
    return [CSRC / name, Path(__file__)] + [CSRC / h if (CSRC / h).exists() else INCLUDE / h for h in headers]


def _up_to_date(out: Path, sources: dict, *more) -> bool:
    """Whether `out` is newer than every source and header; its objects need not
    be there, so that a library that came with the tree is not built again."""
    return _newer(out, [*more, *(i for name, headers in sources.items() for i in _inputs(name, headers))])


def _compile(sources: dict, command, force: bool) -> list:
    """Objects of `sources` by `command`, those that are out of date in parallel."""
    BUILD.mkdir(exist_ok=True)
    objects, todo = [], []
    for name, headers in sources.items():
        obj = BUILD / (name + ".o")
        objects.append(obj)
        if force or not _newer(obj, _inputs(name, headers)):
            todo.append([*command, "-c", CSRC / name, "-o", obj])
    with ThreadPoolExecutor(max_workers=len(sources)) as pool:
        list(pool.map(_run, todo))
    return objects


def build_library(force: bool = False, verbose_ptxas: bool = False) -> Path:
    """nvcc -> libmuon_polar_sm100.so (kernels + C ABI)."""
    out = PKG / LIB_NAME
    if not force and _up_to_date(out, CU_SOURCES):
        return out
    nvcc = _cuda_home() / "bin" / "nvcc"
    cmd = [nvcc, *NVCC_ARCH, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-I", INCLUDE]
    if verbose_ptxas:
        cmd.append("-Xptxas=-v")
    objects = _compile(CU_SOURCES, cmd, force)
    if force or not _newer(out, objects):
        _run([nvcc, *NVCC_ARCH, "-shared", "-Xcompiler", "-fPIC", *objects, "-o", out])
    return out


def build_op(force: bool = False) -> Path:
    """g++ -> _C.so (torch operators), linked to the C ABI library."""
    import torch
    from torch.utils import cpp_extension

    lib = build_library(force=force)
    out = PKG / OP_NAME
    if not force and _up_to_date(out, OP_SOURCES, lib):
        return out
    cuda_home = _cuda_home()
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    includes = cpp_extension.include_paths() + [str(cuda_home / "include"), str(INCLUDE),
                                                sysconfig.get_paths()["include"]]
    objects = _compile(OP_SOURCES, ["g++", "-O2", "-std=c++17", "-fPIC",
                                    f"-D_GLIBCXX_USE_CXX11_ABI={abi}", "-DTORCH_EXTENSION_NAME=_C",
                                    *[f"-I{p}" for p in includes]], force)
    if not force and _newer(out, [*objects, lib]):
        return out
    torch_lib = Path(torch.__file__).resolve().parent / "lib"
    # The operator's inline ATen/c10 helpers call the CUDA runtime: bind them
    # to the same libcudart torch itself loads.
    cudart_dir = torch_lib.parent.parent / "nvidia" / "cuda_runtime" / "lib"
    if (cudart_dir / "libcudart.so.12").exists():
        cudart = [f"-L{cudart_dir}", "-l:libcudart.so.12", f"-Wl,-rpath,{cudart_dir}"]
    else:
        cudart = [f"-L{cuda_home / 'lib64'}", "-lcudart"]
    _run(["g++", "-shared", *objects, "-o", out,
          f"-L{torch_lib}", f"-L{PKG}",
          "-lc10", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-ltorch_cuda",
          "-lmuon_polar_sm100", *cudart,
          "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{torch_lib}"])
    return out


def build_all(force: bool = False) -> None:
    build_library(force=force)
    build_op(force=force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
