"""Builds the B200 LNS libraries in-tree: lib/liblnsb200_<mode>.so, one per
xlns16 summation mode, exactly as the reference builds one tree per
GGML_LNS16_SUM mode (lns-backend/common/lns-common.cmake:24-46).  Every
library also carries the xlns32 (LNSCUDA32) kernels, and the serving kernels
(lnsb_serve.cu), which no summation mode enters: they are compiled once, to an
object that every library links.

    python xlns-ggml-backend_b200/build.py            # all modes
    python xlns-ggml-backend_b200/build.py base sum32 # some
"""
import concurrent.futures
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "lib")

# mode name -> LNSB_SUM_MODE value (csrc/lnsb_arith.cuh)
MODES = {"base": 0, "monte": 1, "monte_bylpvip": 2, "lpvip": 3, "sum32": 4}

SOURCES = ["lnsb_kernels.cu", "lnsb_tables.cpp", "lnsb_graph.cpp"]
SHARED_SOURCES = ["lnsb_serve.cu"]
HEADERS = ["lnsb_arith.cuh", "lnsb_launch.cuh", "lnsb_tables.h", os.path.join(ROOT, "include", "lnsb200.h"),
           os.path.join(ROOT, "include", "lnsb200_graph.h")]


def nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def lib_path(mode):
    return os.path.join(LIB, "liblnsb200_%s.so" % mode)


def _path(name):
    return name if os.path.isabs(name) else os.path.join(CSRC, name)


def _stale(out, sources):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(_path(d)) > t for d in sources + HEADERS)


def _flags(verbose=False):
    return [nvcc()] + (["-Xptxas=-v"] if verbose else []) + [
        "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
        "-Xcompiler", "-fPIC,-ffp-contract=off", "-I", os.path.join(ROOT, "include")]


def _run(what, cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed for %s:\n%s\n%s" % (what, " ".join(cmd), r.stderr))


def build_shared(force=False, verbose=False):
    """the objects that do not depend on the summation mode"""
    outs = []
    os.makedirs(LIB, exist_ok=True)
    for src in SHARED_SOURCES:
        out = os.path.join(LIB, os.path.splitext(src)[0] + ".o")
        if force or _stale(out, [src]):
            _run(src, _flags(verbose) + ["-c", "-o", out + ".tmp", _path(src)])
            os.replace(out + ".tmp", out)
        outs.append(out)
    return outs


def build_mode(mode, force=False, verbose=False, objects=None):
    out = lib_path(mode)
    if not force and not _stale(out, SOURCES + SHARED_SOURCES):
        return out
    objects = objects if objects is not None else build_shared(force, verbose)
    _run("mode " + mode, _flags(verbose) + ["-shared", "-DLNSB_SUM_MODE=%d" % MODES[mode], "-o", out + ".tmp"] +
         [_path(s) for s in SOURCES] + objects)
    os.replace(out + ".tmp", out)
    return out


def build_all(modes=None, force=False):
    modes = list(modes or MODES)
    objects = build_shared(force)
    with concurrent.futures.ThreadPoolExecutor(max_workers=len(modes)) as ex:
        return list(ex.map(lambda m: build_mode(m, force, objects=objects), modes))


if __name__ == "__main__":
    names = [a for a in sys.argv[1:] if not a.startswith("-")]
    for p in build_all(names or None, force="--force" in sys.argv):
        print(p)
