"""Build the B200 kernels in place.

Produces, inside ``sm120_rmsnorm/``:
  * ``libsm120norm_b200.so`` -- the C-ABI library (include/sm120norm_b200.h):
    all CUDA kernels, compiled for sm_100a only, every non-ABI symbol hidden;
  * ``libsm120norm_b200_serving.so`` -- the serving operators
    (include/sm120norm_b200_serving.h), linked against the first;
  * ``_C<ext suffix>``       -- the PyTorch binding (csrc/torch_binding.cpp,
    csrc/serving_binding.cpp), linked against both libraries through an
    ``$ORIGIN`` rpath.

Usage: ``python build.py [--force] [--verbose]`` (``--verbose`` prints
``ptxas -v`` register / spill / shared-memory reports).
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

ROOT = Path(__file__).resolve().parent
REPO = ROOT.parent
PACKAGE = ROOT / "sm120_rmsnorm"
CSRC = ROOT / "csrc"
INCLUDE = REPO / "include"
BUILD = ROOT / "_build"

CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
NVCC = str(CUDA_HOME / "bin" / "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
SHARED_SOURCES = ["device_caches.cu", "cache_args.cu", "tensor_map.cu"]  # in both libraries
NORM_SOURCES = ["runtime.cu", "row_norm.cu", "head_norm_rope.cu", "head_cache.cu", "norm_quant.cu",
                "norm_fp4.cu", "qkv_gemm.cu", *SHARED_SOURCES]
SERVING_SOURCES = ["serving_runtime.cu", "step_plan.cu", "head_mrope.cu", "attention.cu",
                   "attention_mma.cu", "attention_tc.cu",
                   "attention_decode.cu", *SHARED_SOURCES]
BINDING_SOURCES = ["torch_binding.cpp", "serving_binding.cpp"]
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    f"-I{INCLUDE}", f"-I{CSRC}",
]
LIBRARY = PACKAGE / "libsm120norm_b200.so"
SERVING_LIBRARY = PACKAGE / "libsm120norm_b200_serving.so"


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))


def _binding_headers() -> list[Path]:
    return [CSRC / "binding_utils.h", *sorted(INCLUDE.glob("*.h"))]


def _stale(target: Path, sources: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(s.stat().st_mtime > t for s in sources)


def _run(cmd: list[str], verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"command failed ({proc.returncode}): {' '.join(cmd[:3])} ...")
    return proc.stdout + proc.stderr


def _torch_cudart_dirs() -> list[Path]:
    """Directories holding the libcudart.so.12 that PyTorch loads, if any."""
    try:
        import torch
    except ImportError:
        return []
    site = Path(torch.__file__).resolve().parent.parent
    return [d for d in [site / "nvidia" / "cuda_runtime" / "lib"] if (d / "libcudart.so.12").exists()]


def _objects(sources: list[str]) -> list[Path]:
    return [BUILD / (Path(n).stem + ".o") for n in sources]


def _link(target: Path, sources: list[str], extra: list[str], verbose: bool) -> None:
    tmp = BUILD / target.name
    # The CUDA runtime is linked as a shared library so that, inside a
    # PyTorch process, the libraries and PyTorch share one runtime instance
    # (one current device, one set of streams). The rpath prefers the
    # runtime PyTorch ships with, then the toolkit's.
    rpaths = [str(p) for p in _torch_cudart_dirs()] + [str(CUDA_HOME / "lib64")]
    _run([NVCC, *ARCH, "-shared", "-cudart", "shared", *map(str, _objects(sources)), "-o", str(tmp),
          *extra, "-Xlinker", "--exclude-libs,ALL", "-Xlinker", "-Bsymbolic",
          *[f"-Xlinker=-rpath,{r}" for r in rpaths]], verbose)
    os.replace(tmp, target)


def build_library(force: bool = False, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    headers = _headers()
    jobs = []
    for name in dict.fromkeys([*NORM_SOURCES, *SERVING_SOURCES]):
        src = CSRC / name
        obj = BUILD / (Path(name).stem + ".o")
        if force or _stale(obj, [src, *headers]):
            cmd = [NVCC, *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if verbose:
                cmd += ["-Xptxas", "-v"]
            jobs.append(cmd)
    if jobs:
        with ThreadPoolExecutor(max_workers=len(jobs)) as pool:
            for out in pool.map(lambda c: _run(c, verbose), jobs):
                if verbose and out:
                    print(out)
    if force or _stale(LIBRARY, _objects(NORM_SOURCES)):
        _link(LIBRARY, NORM_SOURCES, [], verbose)
    if force or _stale(SERVING_LIBRARY, [*_objects(SERVING_SOURCES), LIBRARY]):
        _link(SERVING_LIBRARY, SERVING_SOURCES,
              [f"-L{PACKAGE}", "-l:" + LIBRARY.name, "-Xlinker", "-rpath,$ORIGIN"], verbose)
    return LIBRARY


def _torch_flags() -> tuple[list[str], list[str]]:
    import torch
    from torch.utils import cpp_extension

    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"],
                str(CUDA_HOME / "include"), str(INCLUDE)]
    flags = [f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             "-DTORCH_EXTENSION_NAME=_C", "-DTORCH_API_INCLUDE_EXTENSION_H"]
    libdirs = cpp_extension.library_paths()
    link = [f"-L{d}" for d in libdirs] + [f"-Wl,-rpath,{d}" for d in libdirs]
    link += ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    return [f"-I{i}" for i in includes] + flags, link


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    suffix = sysconfig.get_config_var("EXT_SUFFIX") or ".so"
    target = PACKAGE / f"_C{suffix}"
    sources = [CSRC / name for name in BINDING_SOURCES]
    headers = _binding_headers()
    if not force and not _stale(target, [*sources, LIBRARY, SERVING_LIBRARY, *headers]):
        return target
    compile_flags, link_flags = _torch_flags()
    BUILD.mkdir(exist_ok=True)
    tmp = BUILD / target.name
    cxx = shutil.which("g++") or "g++"
    objects = [BUILD / (src.stem + ".o") for src in sources]
    jobs = [[cxx, "-O2", "-std=c++17", "-fPIC", *compile_flags, "-c", str(src), "-o", str(obj)]
            for src, obj in zip(sources, objects) if force or _stale(obj, [src, *headers])]
    with ThreadPoolExecutor(max_workers=2) as pool:
        list(pool.map(lambda c: _run(c, verbose), jobs))
    _run([cxx, "-shared", *map(str, objects), "-o", str(tmp), *link_flags, f"-L{PACKAGE}",
          "-l:" + LIBRARY.name, "-l:" + SERVING_LIBRARY.name, "-Wl,-rpath,$ORIGIN"], verbose)
    os.replace(tmp, target)
    return target


def build(force: bool = False, verbose: bool = False) -> None:
    build_library(force, verbose)
    build_binding(force, verbose)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose", action="store_true")
    args = parser.parse_args()
    build(args.force, args.verbose)
    print(f"built {LIBRARY.name} and the _C extension in {PACKAGE}")
