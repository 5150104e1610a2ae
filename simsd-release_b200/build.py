"""Build libsimsd_b200.so (sm_100a) in-tree with nvcc.

    python simsd-release_b200/build.py            # build if any source is newer
    python simsd-release_b200/build.py --force

The library lands next to the Python package (kernels/libsimsd_b200.so), where
kernels/_lib.py loads it, and beside it kernels/_binding.so, the short way from
Python to the serving operators (host code only, against torch's and CPython's headers;
where it cannot be built they are called through ctypes).  nvcc cross-compiles without a
GPU.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import re
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
REPO = PKG.parent
CSRC = PKG / "csrc"
OUT = PKG / "kernels" / "libsimsd_b200.so"
OBJ = PKG / "_build"
BINDING = PKG / "kernels" / "_binding.so"
STAMP = OBJ / "binding.stamp"          # what the binding was built for
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [REPO / "include" / "simsd_b200.h"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else "nvcc"


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or stale(OUT, sources()):
        OBJ.mkdir(exist_ok=True)
        units = sorted(CSRC.glob("*.cu"))
        objs = [str(OBJ / (u.stem + ".o")) for u in units]
        # the translation units compile side by side, then link into one library
        run([[nvcc(), "-O3", "-std=c++17", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC,-O3", "-Xptxas",
              "-v" if verbose else "-O3", "-I", str(REPO / "include"), "-c", "-o", o, str(u)]
             for u, o in zip(units, objs)], verbose)
        run([[nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", str(OUT) + ".tmp", *objs]], verbose)
        os.replace(str(OUT) + ".tmp", OUT)
    try:
        build_binding(force, verbose)
    except (OSError, RuntimeError) as e:
        # the library is complete without it: kernels/_lib.py then calls through ctypes
        BINDING.unlink(missing_ok=True)
        sys.stderr.write(f"{BINDING.name} was not built, the serving operators go through ctypes: {e}\n")
    return OUT


def build_binding(force: bool = False, verbose: bool = False) -> None:
    source = CSRC / "binding.cpp"
    spec = importlib.util.find_spec("torch")
    if spec is None:
        raise RuntimeError("torch is not installed")
    torch = Path(spec.submodule_search_locations[0])
    # torch's C++ interface changes with its version, CPython's with the minor one; _lib.py checks the same text
    version = re.search(r"^__version__ = ['\"](.+)['\"]", (torch / "version.py").read_text(), re.M)
    if version is None:
        raise RuntimeError(f"no version in {torch / 'version.py'}")
    built_for = "torch %s, Python %d.%d" % (version.group(1), *sys.version_info[:2])
    if not (force or stale(BINDING, [source, REPO / "include" / "simsd_b200.h"])
            or not STAMP.exists() or STAMP.read_text() != built_for):
        return
    cuda = Path(nvcc()).resolve().parents[1]
    run([[os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", f'-DSIMSD_BUILT_FOR="{built_for}"',
          "-I", str(REPO / "include"), "-I", sysconfig.get_paths()["include"], "-I", str(torch / "include"),
          "-I", str(torch / "include" / "torch" / "csrc" / "api" / "include"), "-I", str(cuda / "include"),
          "-o", str(BINDING) + ".tmp", str(source), "-L", str(torch / "lib"), "-L", str(cuda / "lib64"),
          "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-lcudart"]], verbose)
    os.replace(str(BINDING) + ".tmp", BINDING)
    STAMP.parent.mkdir(exist_ok=True)
    STAMP.write_text(built_for)


def stale(out: Path, srcs: list[Path]) -> bool:
    return not out.exists() or out.stat().st_mtime < max(p.stat().st_mtime for p in srcs)


def run(cmds: list[list[str]], verbose: bool) -> None:
    procs = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for c in cmds]
    outs = [p.communicate()[0] for p in procs]
    for c, p, out in zip(cmds, procs, outs):
        if p.returncode != 0:
            sys.stderr.write(out)
            raise RuntimeError(f"{Path(c[0]).name} failed ({p.returncode}): {' '.join(c)}")
        if verbose:
            sys.stderr.write(out)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
