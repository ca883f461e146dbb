"""Build the sm_100a CUDA library ``ennx_b200/_lib/libennx_b200.so`` in-tree.

``python -m ennx_b200.build`` (or ``__graft_entry__.build()``) compiles every
``csrc/*.cu`` with nvcc for ``sm_100a`` and links one shared library exporting
the C ABI declared in ``include/ennx_b200.h``, then ``csrc/bindings.cpp`` into
the extension module of the serving operators.  The library needs nvcc alone;
without torch or its C++ headers the module is left out, with a note, and the
serving operators are reached through the C ABI only.  Objects are cached under
``_build/`` and rebuilt when a source or header is newer, the module also when
torch, Python or its command are others than the ones kept beside it.
"""
from __future__ import annotations

import json
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = ROOT / "_build" / "obj"
LIB = PKG / "_lib" / "libennx_b200.so"
BINDINGS = PKG / "_lib" / "ennx_b200_serving.so"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-I", str(ROOT / "include")]


def _headers():
    return list(CSRC.glob("*.cuh")) + list((ROOT / "include").glob("*.h"))


def _compile(src: Path, verbose: bool) -> Path:
    obj = OBJ / (src.stem + ".o")
    newest = max([src.stat().st_mtime] + [h.stat().st_mtime for h in _headers()])
    if obj.exists() and obj.stat().st_mtime >= newest:
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    if verbose and r.stderr:
        print(r.stderr)
    return obj


def bindings_key() -> dict[str, str]:
    """What the extension module's binary interface hangs on, kept beside it."""
    import torch
    return {"torch": torch.__version__, "python": str(sysconfig.get_config_var("SOABI"))}


def _build_bindings() -> None:
    """The torch extension module over the library (host code only), where torch can be built against."""
    try:
        import torch
    except ImportError:
        print("no torch here: the module of the serving operators is not built", file=sys.stderr)
        return
    root, python = Path(torch.__file__).parent, Path(sysconfig.get_paths()["include"])
    if not (root / "include" / "ATen" / "ATen.h").exists() or not (python / "Python.h").exists():
        print("no C++ headers of torch and Python here: the module of the serving operators is not built", file=sys.stderr)
        return
    src = CSRC / "bindings.cpp"
    inc = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", "include",
           Path(NVCC).parents[1] / "include", python]
    made = BINDINGS.with_suffix(f".new{os.getpid()}")  # renamed when whole: ranks may build at once
    # run in ROOT, whose place does not matter: relative paths within it
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-isystem{p}" for p in inc],
           str(src.relative_to(ROOT)), "-L" + str(LIB.parent.relative_to(ROOT)), "-lennx_b200", "-Wl,-rpath,$ORIGIN",
           f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    key = json.dumps({**bindings_key(), "command": cmd}, indent=1)
    stamp = BINDINGS.with_suffix(".key")
    newest = max(p.stat().st_mtime for p in [src, *_headers()])
    if BINDINGS.exists() and BINDINGS.stat().st_mtime >= newest and stamp.exists() and stamp.read_text() == key:
        return
    stamp.unlink(missing_ok=True)
    r = subprocess.run([*cmd, "-o", str(made)], capture_output=True, text=True, cwd=ROOT)
    if r.returncode != 0:
        made.unlink(missing_ok=True)
        raise RuntimeError(f"g++ failed for bindings.cpp:\n{r.stdout}\n{r.stderr}")
    made.replace(BINDINGS)
    stamp.write_text(key)


def build(verbose: bool = False) -> Path:
    OBJ.mkdir(parents=True, exist_ok=True)
    LIB.parent.mkdir(parents=True, exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _build_bindings()
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
