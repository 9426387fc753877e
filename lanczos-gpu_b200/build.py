"""Build liblanczos_b200.so (sm_100a) in-tree.

    python lanczos-gpu_b200/build.py [--force] [--verbose]

Every CUDA source under csrc/ is compiled by nvcc for sm_100a only
(-gencode arch=compute_100a,code=sm_100a) with -lineinfo, then linked into
gpu_eigsh/_lib/liblanczos_b200.so against the static CUDA runtime, so the
library carries no dependency beyond the driver.  Objects go to _build/.
Then csrc/torch/features.cpp, the torch binding of the node-feature operators,
is compiled by g++ against the installed torch and that library into
gpu_eigsh/_lib/_torch_features.so.  Rebuilds only what changed (any header
change rebuilds everything; the binding also for another torch, Python, compiler
or compile command, which _torch_features.json beside it names).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import json
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
OUT_DIR = PKG / "gpu_eigsh" / "_lib"
LIB = OUT_DIR / "liblanczos_b200.so"
TORCH_SRC = CSRC / "torch" / "features.cpp"
TORCH_LIB = OUT_DIR / "_torch_features.so"
TORCH_STAMP = OUT_DIR / "_torch_features.json"   # what the binding was built for
INCLUDE = PKG.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
    "--expt-relaxed-constexpr", "-Xptxas", "-O3", f"-I{INCLUDE}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def host_compiler() -> str:
    """A g++ with a shared libstdc++: one that links its own copy into the binding
    crashes where torch's objects cross between the two."""
    for cand in (shutil.which("g++"), "/usr/bin/g++", os.environ.get("CXX")):
        if cand and Path(cand).exists():
            res = subprocess.run([cand, "-print-file-name=libstdc++.so"], capture_output=True, text=True)
            if os.path.isabs(res.stdout.strip()):
                return cand
    raise RuntimeError("no g++ with a shared libstdc++ found")


def torch_binding_command() -> list[str]:
    """g++ line of the torch binding (torch's own include and library paths)."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cuda = Path(nvcc()).resolve().parents[1]
    inc = [*include_paths(), sysconfig.get_paths()["include"], str(cuda / "include")]
    return [host_compiler(), "-std=c++17", "-O2", "-fPIC", "-shared",
            "-DTORCH_EXTENSION_NAME=_torch_features", "-DTORCH_API_INCLUDE_EXTENSION_H",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in inc),
            str(TORCH_SRC), "-o", str(TORCH_LIB), *(f"-L{p}" for p in library_paths()), "-lc10", "-lc10_cuda", "-ltorch",
            "-ltorch_cpu", "-ltorch_python", f"-L{OUT_DIR}", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"]


def torch_binding_stamp(cmd: list[str]) -> str:
    """What the binding depends on beside its sources: torch's C++ interface changes
    between versions, and a binding for another one does not load, or runs on
    objects of another layout."""
    import sysconfig

    import torch

    compiler = subprocess.run([cmd[0], "--version"], capture_output=True, text=True).stdout.partition("\n")[0]
    return json.dumps({"torch": torch.__version__, "python": sysconfig.get_config_var("SOABI"), "compiler": compiler,
                       "command": [a.replace(str(PKG.parent), ".") for a in cmd]}, indent=1)


def build_torch_binding(force: bool = False, verbose: bool = False) -> None:
    cmd = torch_binding_command()
    stamp = torch_binding_stamp(cmd)
    if (not force and TORCH_LIB.exists() and TORCH_STAMP.exists() and TORCH_STAMP.read_text() == stamp
            and TORCH_LIB.stat().st_mtime >= _newest([TORCH_SRC, *INCLUDE.glob("*.h")])):
        return
    if verbose:
        print(" ".join(cmd), flush=True)
    TORCH_STAMP.unlink(missing_ok=True)   # a build that is cut short leaves none
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed for csrc/torch/features.cpp")
    TORCH_STAMP.write_text(stamp)


def _newest(paths) -> float:
    return max((p.stat().st_mtime for p in paths), default=0.0)


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    hdr_time = _newest(headers)
    cc = nvcc()
    jobs = []
    for src in sources:
        obj = BUILD / (src.stem + ".o")
        stale = force or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, hdr_time)
        if stale:
            flags = NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_verbose else [])
            jobs.append((src, obj, [cc, *flags, "-c", str(src), "-o", str(obj)]))

    def run(job):
        src, obj, cmd = job
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        return src, res

    failed = []
    with cf.ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1)) as ex:
        for src, res in ex.map(run, jobs):
            if res.returncode != 0 or verbose or ptxas_verbose:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                failed.append(src.name)
    if failed:
        raise RuntimeError("nvcc failed for: " + ", ".join(failed))

    objs = [BUILD / (s.stem + ".o") for s in sources]
    if force or jobs or not LIB.exists() or LIB.stat().st_mtime < _newest(objs):
        cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs), "-lpthread", "-ldl",
               "-lrt"]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("link failed")

    build_torch_binding(force, verbose)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas", action="store_true", help="print -Xptxas -v register/smem usage")
    a = ap.parse_args()
    print(build(a.force, a.verbose, a.ptxas))


if __name__ == "__main__":
    main()
