"""Builds libzealot_attn.so in-tree with nvcc for sm_100a.

    python zealot_b200/build.py            # incremental
    python zealot_b200/build.py --force    # rebuild everything

(run as a file, not with -m: importing the package loads the library, which
does not exist yet on a fresh checkout)

Every .cu / .cc file under zealot_b200/csrc is compiled with
-gencode arch=compute_100a,code=sm_100a and linked into
zealot_b200/libzealot_attn.so (static CUDA runtime, no libcuda link: the
driver entry points are resolved at run time, so the library also loads on a
machine without a GPU driver). zealot_b200/calls.c, the Python call path of the
small operators, becomes a module of this CPython beside it, where there are torch
and Python's headers; a host in another language needs only the library.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libzealot_attn.so")
CALLS = os.path.join(HERE, "calls" + sysconfig.get_config_var("EXT_SUFFIX"))  # one for each CPython
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
          "-ccbin", "/usr/bin/g++", f"-I{INCLUDE}", "-I/usr/include"]


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cc")))


def _headers_mtime() -> float:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    hs.append(os.path.join(INCLUDE, "zealot_attn.h"))
    return max(os.path.getmtime(h) for h in hs)


def _compile(src: str, force: bool, verbose_ptxas: bool) -> str:
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    if (not force and os.path.exists(obj) and os.path.getmtime(obj) >= os.path.getmtime(src)
            and os.path.getmtime(obj) >= _headers_mtime()):
        return obj
    cmd = [NVCC, *ARCH, *COMMON, "-c", src, "-o", obj]
    if src.endswith(".cc"):
        cmd[1:1] = ["-x", "cu"]
    if verbose_ptxas and src.endswith(".cu"):
        cmd.append("-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if verbose_ptxas:
        sys.stderr.write(r.stderr)
    return obj


def build(force: bool = False, verbose_ptxas: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, verbose_ptxas), srcs))
    if (force or not os.path.exists(LIB)
            or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs)):
        cmd = [NVCC, *ARCH, "-shared", "-cudart", "static", "-ccbin", "/usr/bin/g++", "-o", LIB,
               *objs, "-ldl", "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _build_calls(force)
    return LIB


def _build_calls(force: bool) -> None:
    src = os.path.join(HERE, "calls.c")
    untagged = os.path.join(HERE, "calls.so")
    if os.path.exists(untagged):  # of a build before the name said which CPython: any would take it
        os.remove(untagged)
    newest = max(os.path.getmtime(src), os.path.getmtime(os.path.join(INCLUDE, "zealot_attn.h")))
    if not force and os.path.exists(CALLS) and os.path.getmtime(CALLS) >= newest:
        return
    torch = importlib.util.find_spec("torch")  # for its tensor exchange header
    python = sysconfig.get_paths()["include"]
    if torch is None or not os.path.exists(os.path.join(python, "Python.h")):
        sys.stderr.write(f"{os.path.basename(CALLS)} is not built (no {'Python.h' if torch else 'torch'} here): the library "
                         "is complete without it, the Python methods of the serving-step operators are not\n")
        return
    cmd = ["gcc", "-O2", "-Wall", "-shared", "-fPIC", f"-I{python}", f"-I{INCLUDE}",
           f"-I{os.path.join(torch.submodule_search_locations[0], 'include')}", src, "-o", CALLS, f"-L{HERE}",
           "-l:libzealot_attn.so", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"gcc failed for {src}:\n{r.stdout}\n{r.stderr}")


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas", action="store_true", help="print -Xptxas -v resource usage")
    a = ap.parse_args()
    print(build(force=a.force, verbose_ptxas=a.ptxas))
