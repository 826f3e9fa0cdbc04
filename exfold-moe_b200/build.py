"""Build libexfold_b200.so in-tree for sm_100a.

    python exfold-moe_b200/build.py [--force] [--verbose]

Each csrc/*.cu is compiled by nvcc (-gencode arch=compute_100a,code=sm_100a, -O3, -lineinfo,
no fast-math, --fmad=false so every float operation is the one written) into
exfold-moe_b200/_build/, then linked into exfold-moe_b200/lib/libexfold_b200.so with the CUDA
runtime linked statically.  Objects are rebuilt only when a source or header is newer.
binding/torch_ops.cpp (host code: autograd nodes over the C ABI) is compiled by g++ against the
installed torch into the Python module lib/libexfold_b200_torch.so, and again when torch or Python change
(lib/libexfold_b200_torch.txt says what it was built for).  The library needs neither torch nor g++: without
them it is built alone.
"""

from __future__ import annotations

import argparse
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = PKG / "_build"
LIB = PKG / "lib" / "libexfold_b200.so"
TORCH_SRC = PKG / "binding" / "torch_ops.cpp"
TORCH_LIB = PKG / "lib" / "libexfold_b200_torch.so"
TORCH_BUILT = TORCH_LIB.with_suffix(".txt")  # what the binding was built for
INCLUDE = ROOT / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--fmad=false", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
              "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def _stale(out: Path, deps: list[Path]) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def torch_command() -> list[str]:
    import torch
    from torch.utils.cpp_extension import include_paths

    libs = Path(torch.__file__).parent / "lib"
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
            "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            f"-I{INCLUDE}", *(arg for p in include_paths() for arg in ("-isystem", p)), "-isystem",
            str(cuda), "-isystem", sysconfig.get_paths()["include"], str(TORCH_SRC), "-o",
            str(TORCH_LIB), f"-L{libs}", "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10",
            "-lc10_cuda", "-ldl", f"-Wl,-rpath,{libs}"]


def torch_built() -> str | None:
    """What a binding built here is for (exfold_b200._lib compares it); None where none can be built."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None or shutil.which("g++") is None:
        return None
    if not (Path(spec.origin).parent / "lib" / "libtorch_cuda.so").exists():
        return None
    version = importlib.metadata.version("torch")
    return f"torch {version}, Python {sys.version_info.major}.{sys.version_info.minor}"


def build_binding(force: bool, run) -> None:
    built = torch_built()
    if built is None:
        print("no torch with CUDA, or no g++: the torch binding is not built, the library is", flush=True)
        return
    if not (force or _stale(TORCH_LIB, [TORCH_SRC, *INCLUDE.glob("*.h")]) or
            not TORCH_BUILT.exists() or TORCH_BUILT.read_text().strip() != built):
        return
    run(torch_command())
    # (a compiler that links its own libstdc++ into the binding would make exceptions of two kinds)
    if "libstdc++.so" not in subprocess.run(["ldd", str(TORCH_LIB)], capture_output=True,
                                            text=True).stdout:
        TORCH_LIB.unlink()
        raise RuntimeError("the torch binding was not linked against the shared libstdc++: use a g++ "
                           "that does")
    TORCH_BUILT.write_text(built + "\n")


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    OBJ.mkdir(parents=True, exist_ok=True)
    LIB.parent.mkdir(parents=True, exist_ok=True)
    headers = _headers()
    sources = sorted(CSRC.glob("*.cu"))
    jobs = []
    for src in sources:
        obj = OBJ / (src.stem + ".o")
        if force or _stale(obj, [src, *headers]):
            cmd = [nvcc(), *ARCH, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o",
                   str(obj)]
            if ptxas_info:
                cmd += ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"build step failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
        if verbose or ptxas_info:
            sys.stdout.write(res.stdout + res.stderr)
        return res

    objs = [OBJ / (s.stem + ".o") for s in sources]
    with ThreadPoolExecutor(max_workers=max(1, min(len(jobs) + 1, os.cpu_count() or 1))) as ex:
        binding = ex.submit(build_binding, force, run)
        list(ex.map(run, jobs))
        if force or _stale(LIB, objs):
            run([nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs)])
        binding.result()
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, ptxas_info=a.ptxas_info))


if __name__ == "__main__":
    main()
