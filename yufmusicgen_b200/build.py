"""Build recipe for ``libyufb200.so`` (sm_100a only) and ``_yuf_torch``, the Python
module that calls it on torch tensors (one per Python; not built where torch is missing,
which the library does without).

Each ``csrc/*.cu`` / ``*.cpp`` file is compiled to an object under
``yufmusicgen_b200/_build/`` (in parallel, skipped when up to date) and linked
into ``yufmusicgen_b200/libyufb200.so`` in the source tree, so the library
travels with the checkout.  ``python -m yufmusicgen_b200.build [-v]``.
"""

from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT_DIR = PKG / "_build"
LIB = PKG / "libyufb200.so"
TORCH_SRC = CSRC / "torch" / "binding.cpp"
TORCH_MODULE = PKG / ("_yuf_torch" + sysconfig.get_config_var("EXT_SUFFIX"))
INCLUDE = PKG.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", str(INCLUDE),
              "--expt-relaxed-constexpr"]
LINK_LIBS = ["-lcudart"]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libyufb200")
    return cand


def _sources():
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, ptxas_verbose: bool) -> tuple[Path, str]:
    obj = OUT_DIR / (src.stem + ".o")
    if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, _headers_mtime()):
        return obj, ""
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    if ptxas_verbose and src.suffix == ".cu":
        cmd += ["-Xptxas", "-v"]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{p.stdout}\n{p.stderr}")
    return obj, p.stderr


def _torch_dir() -> Path | None:
    spec = importlib.util.find_spec("torch")  # found, not imported
    return Path(spec.origin).parent if spec is not None and spec.origin is not None else None


def _compile_torch(torch_dir: Path) -> Path:
    """Compile the torch module's object (it is linked once the library is there)."""
    obj = OUT_DIR / TORCH_MODULE.with_suffix(".o").name
    newest = max(TORCH_SRC.stat().st_mtime, (INCLUDE / "yufb200.h").stat().st_mtime,
                 (torch_dir / "version.py").stat().st_mtime)
    if obj.exists() and obj.stat().st_mtime >= newest:
        return obj
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-I", str(INCLUDE), "-isystem", str(torch_dir / "include"),
           "-isystem", str(torch_dir / "include/torch/csrc/api/include"), "-I", sysconfig.get_paths()["include"],
           "-isystem", str(cuda / "include"), "-c", str(TORCH_SRC), "-o", str(obj)]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"g++ failed on {TORCH_SRC.name}:\n{p.stdout}\n{p.stderr}")
    return obj


def _link_torch(obj: Path, torch_dir: Path) -> None:
    if TORCH_MODULE.exists() and TORCH_MODULE.stat().st_mtime >= obj.stat().st_mtime:
        return
    tmp = TORCH_MODULE.with_suffix(".so.tmp")
    cmd = ["g++", "-shared", "-o", str(tmp), str(obj), "-L", str(PKG), "-lyufb200", "-Wl,-rpath,$ORIGIN",
           "-L", str(torch_dir / "lib"), "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ltorch_python"]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"link of {TORCH_MODULE.name} failed:\n{p.stdout}\n{p.stderr}")
    os.replace(tmp, TORCH_MODULE)


def build(verbose: bool = False, ptxas_verbose: bool = False) -> Path:
    OUT_DIR.mkdir(exist_ok=True)
    srcs = _sources()
    torch_dir = _torch_dir()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        torch_obj = ex.submit(_compile_torch, torch_dir) if torch_dir else None
        results = list(ex.map(lambda s: _compile(s, ptxas_verbose), srcs))
    objs = [o for o, _ in results]
    if verbose:
        for o, log in results:
            if log:
                print(f"--- {o.name}\n{log}", file=sys.stderr)
    newest = max(o.stat().st_mtime for o in objs)
    if not LIB.exists() or LIB.stat().st_mtime < newest:
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), *LINK_LIBS]
        p = subprocess.run(cmd, capture_output=True, text=True)
        if p.returncode != 0:
            raise RuntimeError(f"link failed:\n{p.stdout}\n{p.stderr}")
        os.replace(tmp, LIB)
    if torch_obj is None:
        print("torch not found: _yuf_torch (gated_scan, dropout) is not built", file=sys.stderr)
    else:
        _link_torch(torch_obj.result(), torch_dir)  # its failure is raised here, with the library in place
    return LIB


if __name__ == "__main__":
    v = "-v" in sys.argv
    print(build(verbose=v, ptxas_verbose=v))
