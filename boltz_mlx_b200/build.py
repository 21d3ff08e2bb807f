"""Build libtriattn.so in-tree with nvcc for sm_100a (cross-compiles without a GPU), and the PyTorch binding of
the residual path, _residual.so, with g++ over it.

    python -m boltz_mlx_b200.build            # or: python boltz_mlx_b200/build.py
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libtriattn.so"
RESIDUAL = PKG / "_residual.so"
RESIDUAL_SOURCE = CSRC / "torch_residual.cpp"
SOURCES = ["capi.cu", "kernels_f32.cu", "kernels_tc.cu", "noalloc.cu", "peer.cu", "trimul.cu",
           "residual_capi.cu", "residual_fwd_norm.cu", "residual_fwd_fused.cu", "residual_fwd_fused16.cu",
           "residual_fwd_rows.cu", "residual_bwd_norm.cu", "residual_bwd_fused.cu", "residual_bwd_fused16.cu",
           "dropout_add.cu"]
HEADERS = ["sm100.cuh", "triattn_internal.cuh", "residual.cuh", "residual_fwd.cuh", "residual_bwd.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-shared", "-cudart", "shared",
    "-Xlinker", "-rpath,/usr/local/cuda/lib64",
    "--expt-relaxed-constexpr",
    "-lcublas",
    "--threads", "0",  # the sources compile side by side
]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else "nvcc"


def _older(target: Path, deps: list[Path]) -> bool:
    return not target.exists() or any(d.stat().st_mtime > target.stat().st_mtime for d in deps)


def stale() -> bool:
    return _older(LIB, [CSRC / s for s in SOURCES + HEADERS] + [ROOT / "include" / "triattn.h"])


def built_for(torch) -> str:
    """What the binding is compiled against, as it stands in _residual.so."""
    return f"built for PyTorch {torch.__version__}, Python {sys.version_info.major}.{sys.version_info.minor}"


def residual_stale(torch) -> bool:
    return (_older(RESIDUAL, [RESIDUAL_SOURCE, ROOT / "include" / "triattn.h"])
            or built_for(torch).encode() + b"\0" not in RESIDUAL.read_bytes())


def residual_command(torch) -> list[str]:
    at = Path(torch.__file__).parent
    cuda = Path(nvcc()).resolve().parents[1] if Path(nvcc()).exists() else Path("/usr/local/cuda")
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=_residual",
            "-DTORCH_API_INCLUDE_EXTENSION_H", f'-DRESIDUAL_BUILT_FOR="{built_for(torch)}"', f"-I{at / 'include'}",
            f"-I{at / 'include' / 'torch' / 'csrc' / 'api' / 'include'}", f"-I{cuda / 'include'}",
            f"-I{sysconfig.get_paths()['include']}", f"-I{ROOT / 'include'}", str(RESIDUAL_SOURCE), "-o", str(RESIDUAL),
            f"-L{at / 'lib'}", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10",
            "-lc10_cuda", f"-L{PKG}", "-ltriattn", "-Wl,-rpath,$ORIGIN"]


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout or r.stderr):
        print(r.stdout, r.stderr)


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> Path:
    if force or stale():
        _run([nvcc(), *NVCC_FLAGS, *(extra or []), "-I", str(ROOT / "include"), "-I", str(CSRC),
              "-o", str(LIB), *[str(CSRC / s) for s in SOURCES]], verbose)
    try:
        import torch
    except ImportError:  # the C library needs none
        print(f"PyTorch is not installed: {RESIDUAL.name}, its binding, is left out")
        return LIB
    if force or residual_stale(torch):
        _run(residual_command(torch), verbose)
    return LIB


if __name__ == "__main__":
    extra = sys.argv[1:]
    print(build(force=True, verbose=True, extra=extra))
