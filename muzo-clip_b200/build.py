"""Build the sm_100a shared library behind muzo_clip_b200.

Compiles every ``csrc/*.cu`` and ``csrc/*.cpp`` with nvcc for ``sm_100a`` (nvcc cross-compiles,
no GPU is needed) and links them into ``muzo_clip_b200/libmuzo_b200.so`` next to the Python
package, where ``muzo_clip_b200._lib`` loads it. Objects go to ``_build/`` and are rebuilt only
when a source or header is newer.

``csrc/binding/native.cpp`` becomes the Python module ``muzo_clip_b200/_native*.so`` (g++ against the
installed torch's headers).

Usage: ``python build.py [--force] [--jobs N]``
"""

from __future__ import annotations

import argparse
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
INCLUDE = ROOT / "include"
BUILD = HERE / "_build"
OUT = HERE / "muzo_clip_b200" / "libmuzo_b200.so"
NATIVE_SRC = CSRC / "binding" / "native.cpp"
NATIVE = HERE / "muzo_clip_b200" / f"_native{sysconfig.get_config_var('EXT_SUFFIX')}"

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", f"-I{INCLUDE}", f"-I{CSRC}"]


def _sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h")))


def _compile(src: Path, force: bool) -> Path:
    obj = BUILD / (src.name + ".o")
    newest_dep = max([src.stat().st_mtime] + [h.stat().st_mtime for h in _headers()])
    if not force and obj.exists() and obj.stat().st_mtime >= newest_dep:
        return obj
    cmd = [NVCC, *ARCH, *COMMON, "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cpp":
        cmd = [NVCC, *COMMON, "-x", "c++", "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    return obj


def build_native(force: bool = False) -> Path:
    """The Python module over torch tensors; rebuilt when its source, the C header or torch change."""
    import torch
    from torch.utils import cpp_extension

    stamp = BUILD / "native.torch"
    newest = max(p.stat().st_mtime for p in (NATIVE_SRC, INCLUDE / "muzo_b200.h"))
    if not force and NATIVE.exists() and NATIVE.stat().st_mtime >= newest and stamp.exists() \
            and stamp.read_text() == torch.__version__:
        return NATIVE
    cuda = Path(NVCC).resolve().parent.parent
    includes = [*cpp_extension.include_paths(), str(cuda / "include"), str(INCLUDE), sysconfig.get_path("include")]
    libs = Path(torch.__file__).parent / "lib"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_native",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-isystem{p}" for p in includes], str(NATIVE_SRC), "-o", str(NATIVE), f"-L{libs}", "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {NATIVE_SRC.name}:\n{res.stdout}\n{res.stderr}")
    stamp.write_text(torch.__version__)
    return NATIVE


def build(force: bool = False, jobs: int | None = None) -> Path:
    BUILD.mkdir(exist_ok=True)
    srcs = _sources()
    with ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 1)) as ex:
        native = ex.submit(build_native, force)
        objs = list(ex.map(lambda s: _compile(s, force), srcs))
        native.result()
    newest = max(o.stat().st_mtime for o in objs)
    if force or not OUT.exists() or OUT.stat().st_mtime < newest:
        cmd = [NVCC, *ARCH, "-shared", "-cudart", "static", "-o", str(OUT), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    return OUT


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args()
    out = build(force=args.force, jobs=args.jobs)
    print(out)
    return 0


if __name__ == "__main__":
    sys.exit(main())
