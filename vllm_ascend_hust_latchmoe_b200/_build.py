"""Build liblatchmoe_b200.so in-tree with nvcc for sm_100a (B200).

The library is a plain C-ABI shared object (no torch types cross its boundary); the
package loads it with ctypes. ``_decoder_ops.so`` beside it is the decoder operators' Python
binding (host code only: torch tensors in, calls of the C ABI out) and is built for one torch
and one Python. The library needs nvcc alone and is built first, with or without the binding.
Both are built next to this file so that they travel with the source tree; nothing is installed
into site-packages.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_ROOT = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
INCLUDE = REPO_ROOT / "include"
LIB_NAME = "liblatchmoe_b200.so"
LIB_PATH = PKG_DIR / LIB_NAME

BINDING_SRC = CSRC / "binding" / "decoder_ops.cpp"
BINDING_PATH = PKG_DIR / "_decoder_ops.so"

NVCC_FLAGS = (
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-shared",
    "-Xcompiler",
    "-fPIC",
)


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _inputs_mtime() -> float:
    paths = _sources() + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    return max(p.stat().st_mtime for p in paths)


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return str(cand)
    raise RuntimeError("nvcc not found: set NVCC or put /usr/local/cuda/bin on PATH")


def _run(what: str, cmd: list[str], out: Path, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{what} failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    os.replace(cmd[cmd.index("-o") + 1], out)


def binding_key() -> str:
    """What the binding is built for; compiled into it."""
    import torch

    return (f"lm-binding {sys.implementation.cache_tag} torch {torch.__version__} "
            f"cxx11 {int(torch.compiled_with_cxx11_abi())}")


def binding_is_current() -> bool:
    """Built from the present sources for this torch and this Python."""
    if not BINDING_PATH.exists():
        return False
    newest = max(p.stat().st_mtime for p in (BINDING_SRC, *INCLUDE.glob("*.h")))
    return BINDING_PATH.stat().st_mtime >= newest and binding_key().encode() in BINDING_PATH.read_bytes()


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile the decoder operators' binding with the host compiler (skipped when up to date).
    A binding that is out of date is removed first: without one, its operators say so."""
    if not force and binding_is_current():
        return BINDING_PATH
    import torch

    BINDING_PATH.unlink(missing_ok=True)
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parents[1]
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f'-DLM_BUILT_FOR="{binding_key()}"', f"-I{INCLUDE}",
           f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}",
           f"-I{sysconfig.get_paths()['include']}", f"-I{cuda / 'include'}",
           "-o", str(BINDING_PATH.with_suffix(".so.tmp")), str(BINDING_SRC),
           f"-L{root / 'lib'}", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ltorch_python"]
    _run("the binding's build", cmd, BINDING_PATH, verbose)
    return BINDING_PATH


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile every .cu under csrc/ into one shared library (skipped when up to date)."""
    if not force and LIB_PATH.exists() and LIB_PATH.stat().st_mtime >= _inputs_mtime():
        return LIB_PATH
    tmp = LIB_PATH.with_suffix(".so.tmp")
    _run("nvcc", [nvcc_path(), *NVCC_FLAGS, f"-I{INCLUDE}", "-o", str(tmp), *map(str, _sources())],
         LIB_PATH, verbose)
    return LIB_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """The library, and then the binding where it can be built (a warning where it cannot: no host
    compiler, no headers). Returns the library's path."""
    path = build_library(force, verbose)
    try:
        build_binding(force, verbose)
    except (ImportError, OSError, RuntimeError) as e:
        warnings.warn(f"{BINDING_PATH.name} is not built, decoder_ops will refuse its calls: {e}")
    return path


if __name__ == "__main__":
    print(build(force=True, verbose=True))
