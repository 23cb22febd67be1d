"""Builds libskm_b200.so in-tree with nvcc for sm_100a.  Run as `python superkmeans_b200/build.py` (by path: importing the package needs the library).

`_ops_calls`, the short cuts of ops.py into that library, is built beside it where torch and Python's headers are there; ops.py works without,
and so does this where it cannot be compiled or linked (a torch without CUDA).  It is made for one torch and one Python, whose names it carries: it is
built again for others, and ops.py leaves one that was built for others alone.

Every source file is compiled to an object of its own (in parallel, and only when it or a header changed), then the
objects are linked into the shared library.  `-v` prints what ptxas reports (registers, spills, shared memory)."""
from __future__ import annotations

import importlib.util
import os
import runpy
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJDIR = os.path.join(HERE, "build")
SOURCES = ["memory.cu", "host_copy.cu", "phase_timers.cu", "kernels.cu", "kernels_pruned_dense.cu", "kernels_tc.cu", "kernels_tc_sparse.cu", "kernels_tc_rotate.cu", "kernels_tc_rotate_half.cu", "kernels_first_test.cu", "kernels_chain.cu", "kernels_walk.cu", "kernels_topk.cu", "kernels_replay.cu", "rotation_matrix.cu", "exact_assign.cu", "direct_assign.cu", "rows_group.cu", "rows_move.cu", "rows_unaligned.cu", "rows_sum.cu", "product_8bit.cu", "engine.cu", "engine_fine.cu",
           "comm_nccl.cu", "noalloc.cu", "abi.cu"]
HEADERS = ["common.cuh", "device_utils.cuh", "gemm_simt.cuh", "tc_ptx.cuh", "kernels_tc.cuh", "rows.h", "rows_access.cuh", "noalloc.h", "engine.h", "engine_buffers.h", "host_copy.h", "phase_timers.h", "exact_assign.h", "host_logic.h", "comm_nccl.h",
           os.path.join("..", "..", "include", "skm_b200.h")]
OUTPUT = os.path.join(HERE, "libskm_b200.so")
CALLS_SOURCE = os.path.join(CSRC, "ops_calls.cpp")
CALLS_OUTPUT = os.path.join(HERE, "_ops_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
CALLS_BUILT_FOR = os.path.join(HERE, "_ops_calls.built_for")


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _sources():
    return [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]


def _newest_header() -> float:
    paths = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.abspath(__file__)]
    return max(os.path.getmtime(p) for p in paths if os.path.exists(p))


def needs_build() -> bool:
    if not os.path.exists(OUTPUT):
        return True
    t = os.path.getmtime(OUTPUT)
    if _newest_header() > t:
        return True
    return any(os.path.getmtime(os.path.join(CSRC, s)) > t for s in _sources())


def _compile_one(nvcc: str, src: str, verbose: bool):
    obj = os.path.join(OBJDIR, os.path.splitext(src)[0] + ".o")
    cmd = [
        nvcc, "-std=c++17", "-O3", "-lineinfo", "-c",
        "-gencode", "arch=compute_100a,code=sm_100a",
        "-ccbin", "/usr/bin/g++",
        "-Xcompiler", "-fPIC,-fopenmp,-O3,-Wall,-Wno-unknown-pragmas",
    ]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += [os.path.join(CSRC, src), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    return src, obj, res


def _torch_dir():
    found = importlib.util.find_spec("torch")
    return None if found is None else os.path.dirname(found.origin)


def calls_built_for(torch_dir: str) -> str:
    """The torch and the Python that the short cuts are made for (ops.py says the same of those that it runs with)."""
    version = runpy.run_path(os.path.join(torch_dir, "version.py"))
    return f"torch {version['__version__']}, CUDA {version['cuda']}, {sysconfig.get_config_var('SOABI')}"


def _stale_calls(built_for: str) -> bool:
    if not os.path.exists(CALLS_OUTPUT) or not os.path.exists(CALLS_BUILT_FOR):
        return True
    with open(CALLS_BUILT_FOR) as f:
        if f.read() != built_for:
            return True
    header = os.path.join(CSRC, "..", "..", "include", "skm_b200.h")
    return max(os.path.getmtime(CALLS_SOURCE), os.path.getmtime(header)) > os.path.getmtime(CALLS_OUTPUT)


def build_calls(force: bool = False) -> None:
    """The short cuts between torch tensors and the library (needs the library)."""
    include = sysconfig.get_paths()["include"]
    torch_dir = _torch_dir()
    if torch_dir is None or not os.path.exists(os.path.join(include, "Python.h")):
        sys.stderr.write("torch or Python.h is missing: ops.py goes without its short cuts\n")
        return
    built_for = calls_built_for(torch_dir)
    if not force and not _stale_calls(built_for):
        return
    for old in (CALLS_OUTPUT, CALLS_BUILT_FOR, os.path.join(HERE, "_ops_calls.so")):   # (the last: of a build that named no Python)
        if os.path.exists(old):
            os.remove(old)
    try:
        import torch

        cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
        cmd = ["/usr/bin/g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f'-DSKM_BUILT_FOR="{built_for}"',
               f"-I{include}", f"-I{torch_dir}/include", f"-I{torch_dir}/include/torch/csrc/api/include",
               f"-I{cuda}/include", CALLS_SOURCE, "-o", CALLS_OUTPUT, f"-L{torch_dir}/lib", "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda", f"-L{HERE}", "-lskm_b200",
               "-Wl,-rpath,$ORIGIN"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        failed = res.stdout + res.stderr if res.returncode != 0 else None
    except (ImportError, OSError) as e:
        failed = f"{e}\n"
    if failed is not None:
        sys.stderr.write(failed + "compiling ops_calls.cpp failed: ops.py goes without its short cuts\n")
        return
    with open(CALLS_BUILT_FOR, "w") as f:
        f.write(built_for)


def build(force: bool = False, verbose: bool = False) -> str:
    if force or verbose or needs_build():
        build_library(force, verbose)
    build_calls(force)
    return OUTPUT


def build_library(force: bool, verbose: bool) -> None:
    nvcc = _nvcc()
    os.makedirs(OBJDIR, exist_ok=True)
    hdr_t = _newest_header()
    todo, objs = [], []
    for src in _sources():
        obj = os.path.join(OBJDIR, os.path.splitext(src)[0] + ".o")
        objs.append(obj)
        stale = force or verbose or not os.path.exists(obj) or os.path.getmtime(obj) < max(hdr_t, os.path.getmtime(os.path.join(CSRC, src)))
        if stale:
            todo.append(src)
    failed = False
    with ThreadPoolExecutor(max_workers=max(1, min(len(todo), os.cpu_count() or 1))) as pool:
        for src, _obj, res in pool.map(lambda s: _compile_one(nvcc, s, verbose), todo):
            if res.returncode != 0:
                sys.stderr.write(f"--- {src}\n" + res.stdout + res.stderr)
                failed = True
            elif verbose or res.stderr.strip():
                sys.stderr.write(f"--- {src}\n" + res.stdout + res.stderr)
    if failed:
        raise RuntimeError("nvcc failed")
    link = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-ccbin", "/usr/bin/g++", "-cudart", "static", "-Xcompiler", "-fPIC"] + objs + ["-o", OUTPUT, "-lgomp", "-ldl"]
    res = subprocess.run(link, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("link failed")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
