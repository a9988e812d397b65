"""Build the in-tree CUDA library ``crukx_sync_b200/libcrukx_b200.so`` for sm_100a with nvcc, and the
torch side of trainer.py's calls, ``crukx_sync_b200/_glue.so``, with g++.

    python -m crukx_sync_b200.build [--force] [--verbose]

Objects go to ``crukx_sync_b200/_build/``; a file is recompiled when it or any header is newer
than its object.  The library exports the C ABI declared in ``include/crukx_b200.h``.  The torch side is
compiled again for another torch or Python too; where it cannot be (no headers of theirs), that is
reported and the library stands: the codec does without it, and trainer.py's calls say what is missing.
"""

from __future__ import annotations

import concurrent.futures
import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libcrukx_b200.so")
GLUE_SRC = os.path.join(CSRC, "glue", "torch_glue.cpp")
GLUE = os.path.join(HERE, "_glue.so")
GLUE_BUILT = os.path.join(BUILD, "glue.built")   # what it was built for
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3", "-I", os.path.join(ROOT, "include"),
         "--expt-relaxed-constexpr"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the crukx_sync_b200 CUDA library cannot be built")


def cxx() -> str:
    return os.environ.get("CXX") or shutil.which("g++") or "g++"


def _headers():
    return glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(ROOT, "include", "*.h"))


def glue_command(out: str) -> list[str]:
    spec = importlib.util.find_spec("torch")   # (found, not imported: that takes a while)
    if spec is None:
        raise RuntimeError("torch not found")
    torch = os.path.dirname(spec.origin)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    include = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    return [cxx(), "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_glue", "-DTORCH_API_INCLUDE_EXTENSION_H",
            *[x for d in include for x in ("-I", d)], GLUE_SRC, "-o", out, "-L", HERE, "-l:libcrukx_b200.so",
            "-L", os.path.join(torch, "lib"), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
            "-Wl,-rpath,$ORIGIN"]


def build_glue(run, force: bool = False) -> None:
    built_for = f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}\n"
    newest = max(os.path.getmtime(GLUE_SRC), os.path.getmtime(os.path.join(ROOT, "include", "crukx_b200.h")))
    if not force and os.path.exists(GLUE) and os.path.getmtime(GLUE) >= newest and os.path.exists(GLUE_BUILT):
        with open(GLUE_BUILT) as f:
            if f.read() == built_for:
                return
    if os.path.exists(GLUE):
        os.remove(GLUE)   # not left behind when the compiler fails
    tmp = GLUE + ".tmp"
    run(glue_command(tmp))
    os.replace(tmp, GLUE)
    with open(GLUE_BUILT, "w") as f:
        f.write(built_for)


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))
    newest_header = max((os.path.getmtime(h) for h in _headers()), default=0.0)
    cc = nvcc()
    jobs = []
    objs = []
    for src in srcs:
        obj = os.path.join(BUILD, os.path.basename(src) + ".o")
        objs.append(obj)
        stale = force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), newest_header)
        if stale:
            cmd = [cc, *ARCH, *FLAGS, *(extra or []), "-c", src, "-o", obj]
            if src.endswith(".cpp"):
                cmd = [cxx(), "-O3", "-std=c++17", "-fPIC", "-Wall", "-I", os.path.join(ROOT, "include"),
                       "-c", src, "-o", obj]
            jobs.append(cmd)

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"compiler failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, flush=True)

    with concurrent.futures.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        list(ex.map(run, jobs))
    if jobs or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        tmp = LIB + ".tmp"
        run([cc, *ARCH, "-shared", "-o", tmp, *objs, "-lcudart"])
        os.replace(tmp, LIB)
    try:
        build_glue(run, force)
    except (RuntimeError, OSError, importlib.metadata.PackageNotFoundError) as exc:
        print(f"crukx_sync_b200: _glue.so was not built, trainer.py's calls will not run: {exc}", file=sys.stderr, flush=True)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(LIB)
