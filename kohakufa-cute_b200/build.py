"""Builds libkfa.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a.

    python kohakufa-cute_b200/build.py [--force] [--phases]

The shared library is written next to the Python package as ``kohakufa_cute/libkfa.so``.
``--phases`` builds a second library, ``kohakufa_cute/libkfa_phases.so``, whose pipeline kernels record
how many cycles each role of one CTA spends in each phase of its loop (see ``csrc/phase_clock.cuh``;
``phase_profile.py`` runs it and prints the table).  The ordinary library carries none of that code.
"""

import hashlib
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "kohakufa_cute")
OBJ_DIR = os.path.join(HERE, "build")
LIB = os.path.join(OUT_DIR, "libkfa.so")
SOURCES = ["kfa_api.cu", "general_kernels.cu", "neighborhood_kernels.cu", "pipeline_forward.cu", "decode_forward.cu",
           "pipeline_backward.cu", "wide_head.cu", "na_pipeline.cu", "tensor_map.cu", "static_scratch.cu", "wait_probe.cu", "center_keys_cluster.cu",
           "quantized_cache.cu", "cache_attention.cu", "window_decode.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
              "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "-Wno-deprecated-gpu-targets"]


def _nvcc():
    return os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc")


def _digest(paths, flags):
    h = hashlib.sha256()
    for path in sorted(paths):
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(" ".join(flags).encode())
    return h.hexdigest()


def sources():
    return [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]


def build(force=False, verbose=True, phases=False):
    flags = NVCC_FLAGS + (["-DKFA_PHASES=1"] if phases else [])
    obj_dir = OBJ_DIR + ("_phases" if phases else "")
    lib = LIB.replace("libkfa.so", "libkfa_phases.so") if phases else LIB
    os.makedirs(obj_dir, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh", ".inl"))]
    headers.append(os.path.join(os.path.dirname(HERE), "include", "kfa.h"))
    objects, jobs = [], []
    for src in sources():
        path = os.path.join(CSRC, src)
        obj = os.path.join(obj_dir, src.replace(".cu", ".o"))
        stamp = obj + ".sha"
        digest = _digest([path] + headers, flags)
        objects.append(obj)
        fresh = os.path.exists(obj) and os.path.exists(stamp) and open(stamp).read() == digest
        if force or not fresh:
            jobs.append((path, obj, stamp, digest))

    def compile_one(job):
        path, obj, stamp, digest = job
        cmd = [_nvcc(), *flags, "-c", path, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        with open(stamp, "w") as f:
            f.write(digest)

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as pool:
        list(pool.map(compile_one, jobs))
    if jobs or force or not os.path.exists(lib):
        cmd = [_nvcc(), "-shared", "-o", lib, *objects, "-lcudart_static", "-ldl", "-lpthread", "-lrt",
               "-Wno-deprecated-gpu-targets"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    if not phases:
        build_records(force, verbose)
        build_calls(force, verbose)
    return lib


def _compile_module(target, cmd, stamp, digest, force, verbose):
    """Compiles an optional module unless it is there as `digest` describes it; ``None``, and no module of other sources or
    another torch left behind, where that fails."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    if force or not os.path.exists(target) or not os.path.exists(stamp) or open(stamp).read() != digest:
        if verbose:
            print(" ".join(cmd + ["-o", target]), flush=True)
        try:
            subprocess.check_call(cmd + ["-o", target])
        except (OSError, subprocess.CalledProcessError) as error:
            return _left_out(target, error)
        with open(stamp, "w") as f:
            f.write(digest)
    return target


def _left_out(target, reason):
    print(f"left out: {target} ({reason})", flush=True)
    if os.path.exists(target):
        os.remove(target)
    return None


def build_records(force=False, verbose=True):
    """The optional CPython module that packs tensor records (``csrc/fast_records.c``), or ``None`` without Python's
    headers or a compiler for them: the binding then packs them itself, with the same results."""
    include = sysconfig.get_paths()["include"]
    source = os.path.join(CSRC, "fast_records.c")
    header = os.path.join(os.path.dirname(HERE), "include", "kfa.h")
    target = os.path.join(OUT_DIR, "_fast_records" + sysconfig.get_config_var("EXT_SUFFIX"))
    if not os.path.exists(os.path.join(include, "Python.h")):
        return _left_out(target, "no Python.h")
    cmd = [os.environ.get("CC", "gcc"), "-O2", "-std=c11", "-Wall", "-Wextra", "-shared", "-fPIC", "-I", include, source]
    return _compile_module(target, cmd, os.path.join(OBJ_DIR, "fast_records.sha"), _digest([source, header], cmd), force, verbose)


def build_calls(force=False, verbose=True):
    """The optional torch module that serves plain window and cache calls in one step (``csrc/fast_calls.cpp``), or
    ``None`` without the headers it needs, or where this torch's do not compile here: the Python layer then serves
    them, with the same results."""
    include = sysconfig.get_paths()["include"]
    spec = importlib.util.find_spec("torch")
    home = os.path.dirname(spec.origin) if spec and spec.origin else ""
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(_nvcc()) or _nvcc()))), "include")
    target = os.path.join(OUT_DIR, "_fast_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
    version = os.path.join(home, "version.py")
    needed = (os.path.join(include, "Python.h"), os.path.join(home, "include", "c10", "cuda", "CUDAStream.h"),
              os.path.join(cuda, "cuda_runtime_api.h"), version)
    missing = [path for path in needed if not os.path.exists(path)]
    if missing:
        return _left_out(target, f"no {missing[0]}")
    source = os.path.join(CSRC, "fast_calls.cpp")
    header = os.path.join(os.path.dirname(HERE), "include", "kfa.h")
    # the module belongs to one torch, whose version it carries: the binding uses it with no other
    with open(version) as f:
        torch_version = re.search(r"""^__version__ = ['"]([^'"]+)""", f.read(), re.MULTILINE)
    if torch_version is None:
        return _left_out(target, "torch has no version")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-Wall", "-shared", "-fPIC", "-fvisibility=hidden", "-I", include,
           f'-DKFA_TORCH_VERSION="{torch_version.group(1)}"']
    for path in (os.path.join(home, "include"), os.path.join(home, "include", "torch", "csrc", "api", "include"), cuda):
        cmd += ["-isystem", path]
    cmd += [source, "-L", os.path.join(home, "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda"]
    return _compile_module(target, cmd, os.path.join(OBJ_DIR, "fast_calls.sha"), _digest([source, header, version], cmd), force,
                           verbose)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, phases="--phases" in sys.argv))
