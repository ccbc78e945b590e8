"""Build the HIP libraries (gfx950) in-tree with hipcc.

Usage: ``python isa-_amd/csrc/build.py`` (also called by ``__graft_entry__.build()``).
Each library lands next to its loader: ``libisa_ekv_hip.so`` in ``isa/kernels/transformer_ffn/``, which
loads it with ctypes; ``libisa_block_hip.so`` in ``isa/kernels/transformer_block/`` with ``_binding.so``,
torch's binding to it, a module that the package imports.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG_ROOT = CSRC.parent
REPO = PKG_ROOT.parent
SOURCES = [CSRC / "ekv_lut.hip"]
INCLUDE = REPO / "include"
OUT = PKG_ROOT / "isa" / "kernels" / "transformer_ffn" / "libisa_ekv_hip.so"
BLOCK_SOURCES = [CSRC / f"block_{name}.hip" for name in ("api", "norm", "attention", "attention_backward", "loss")]
# products keep their sums in ordinary registers, which the softmax between two products works on: with
# accumulation registers every one of them is moved there and back
BLOCK_FLAGS = ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]
BLOCK_OUT = PKG_ROOT / "isa" / "kernels" / "transformer_block" / "libisa_block_hip.so"
BINDING_SOURCE = CSRC / "block_torch.cpp"
BINDING_OUT = BLOCK_OUT.with_name("_binding.so")
ARCH = os.environ.get("ISA_EKV_OFFLOAD_ARCH", "gfx950")

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    # packed FP32 ops stay off on this pool; hipcc -O3 would otherwise form them
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found: set HIPCC or install ROCm")


def _run(cmd: list, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")


def _ekv(verbose: bool) -> None:
    tmp = OUT.with_suffix(".so.tmp")
    _run([hipcc(), *HIPCC_FLAGS, f"-I{INCLUDE}", "-o", str(tmp), *map(str, SOURCES)], verbose)
    os.replace(tmp, OUT)


def _block(verbose: bool, pool: ThreadPoolExecutor) -> None:
    compile_flags = [f for f in HIPCC_FLAGS if f != "-shared"]
    tmp = BLOCK_OUT.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory() as work:
        objects = [str(Path(work) / f"{src.stem}.o") for src in BLOCK_SOURCES]
        jobs = [pool.submit(_run, [hipcc(), *compile_flags, *BLOCK_FLAGS, f"-I{INCLUDE}", "-c", "-o", obj, str(src)], verbose)
                for src, obj in zip(BLOCK_SOURCES, objects)]
        for job in jobs:
            job.result()
        _run([hipcc(), *HIPCC_FLAGS, "-o", str(tmp), *objects], verbose)
    os.replace(tmp, BLOCK_OUT)


def _binding_object(obj: Path, verbose: bool) -> None:
    import torch
    from torch.utils.cpp_extension import include_paths

    # the HIP headers' own switch, and torch's: which GPU runtime its headers stand for
    flags = ["-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1"]
    rocm = Path(hipcc()).resolve().parents[1] / "include"
    includes = [f"-I{INCLUDE}", *(f"-isystem{p}" for p in (*include_paths(), sysconfig.get_paths()["include"], rocm))]
    _run(["g++", "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *flags, *includes, "-c", "-o", str(obj), str(BINDING_SOURCE)], verbose)


def _link_binding(obj: Path, verbose: bool) -> None:
    import torch

    lib = Path(torch.__file__).resolve().parent / "lib"
    tmp = BINDING_OUT.with_suffix(".so.tmp")
    _run(["g++", "-shared", "-o", str(tmp), str(obj), f"-L{BLOCK_OUT.parent}", "-lisa_block_hip", f"-L{lib}", "-lc10",
          "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], verbose)
    os.replace(tmp, BINDING_OUT)


def build(verbose: bool = False) -> Path:
    """Compile the libraries and the binding, side by side; returns the projection's library."""
    with tempfile.TemporaryDirectory() as work, ThreadPoolExecutor(max_workers=2 + len(BLOCK_SOURCES)) as pool:
        obj = Path(work) / "binding.o"
        others = [pool.submit(_ekv, verbose), pool.submit(_binding_object, obj, verbose)]
        _block(verbose, pool)
        for job in others:
            job.result()
        _link_binding(obj, verbose)
    return OUT


if __name__ == "__main__":
    path = build(verbose=True)
    print(f"built {path}\nbuilt {BLOCK_OUT}\nbuilt {BINDING_OUT}")
    sys.exit(0)
