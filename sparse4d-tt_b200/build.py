"""Build ``lib/libs4d_dfa.so`` (the C ABI of ``include/s4d_dfa.h``) and ``lib/libs4d_decoder.so``
(``include/s4d_decoder.h``) for sm_100a with nvcc, and the Python module of the latter's calls with g++.

    python sparse4d-tt_b200/build.py [--verbose-ptxas]

The libraries are built in-tree so that they travel with the repository; nothing is installed.
"""
from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_DIR = os.path.join(PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libs4d_dfa.so")
SOURCES = ["capi.cu", "kps_project.cu", "dfa_gather.cu", "kps_noalloc.cu", "linear_tc.cu", "camera_encoder.cu", "pack_maps.cu",
           "instance_bank.cu", "peer.cu", "layer_norm.cu"]
# The decoder's operators: each (source, defines) is compiled by itself, several at a time.
DECODER_LIB_PATH = os.path.join(LIB_DIR, "libs4d_decoder.so")
DECODER_SOURCES = [("decoder_capi.cu",), ("decoder_norm.cu",), ("decoder_attention.cu",),
                   ("decoder_attention_forward.cu", "-DS4D_HEAD_DIM=64"),
                   ("decoder_attention_forward.cu", "-DS4D_HEAD_DIM=128"),
                   ("decoder_attention_backward.cu", "-DS4D_HEAD_DIM=64"),
                   ("decoder_attention_backward.cu", "-DS4D_HEAD_DIM=128")]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def _run(cmd, what: str, verbose_ptxas: bool) -> None:
    if verbose_ptxas:
        cmd = [cmd[0], "-Xptxas", "-v", *cmd[1:]]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed building {what}")
    if verbose_ptxas:
        sys.stdout.write(res.stderr)


def build_decoder(verbose_ptxas: bool = False, force: bool = False) -> str:
    """``libs4d_decoder.so`` and the module of its calls; objects newer than their source and every header are kept."""
    obj_dir = os.path.join(LIB_DIR, "obj")
    headers = [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith(".cuh")]
    headers += [os.path.join(INCLUDE, h) for h in os.listdir(INCLUDE)] + [os.path.abspath(__file__)]
    newest_header = max(os.path.getmtime(h) for h in headers)
    os.makedirs(obj_dir, exist_ok=True)
    flags = [*ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
             "-I", INCLUDE, "-I", CSRC]
    objs, jobs = [], []
    for name, *defs in DECODER_SOURCES:
        src, obj = os.path.join(CSRC, name), os.path.join(obj_dir, "_".join([name[:-3], *(d.split("=")[-1] for d in defs)])
                                                          + ".o")
        objs.append(obj)
        if force or verbose_ptxas or not os.path.exists(obj) or os.path.getmtime(obj) < max(newest_header,
                                                                                            os.path.getmtime(src)):
            jobs.append((src, obj, defs))
    with concurrent.futures.ThreadPoolExecutor(max(1, os.cpu_count() or 1)) as pool:
        for f in [pool.submit(_run, [nvcc_path(), *flags, *defs, "-c", "-o", obj, src], os.path.basename(src),
                              verbose_ptxas) for src, obj, defs in jobs]:
            f.result()
    if jobs or not os.path.exists(DECODER_LIB_PATH) or any(os.path.getmtime(o) > os.path.getmtime(DECODER_LIB_PATH)
                                                           for o in objs):
        _run([nvcc_path(), *ARCH_FLAGS, "--shared", "-o", DECODER_LIB_PATH + ".tmp", *objs, "-lcudart"],
             "libs4d_decoder.so", False)
        os.replace(DECODER_LIB_PATH + ".tmp", DECODER_LIB_PATH)
    build_calls(force)
    return DECODER_LIB_PATH


def calls_path() -> str:
    """Where the module of the decoder's calls is for this Python and torch, whose internals it is compiled against: one
    that was built for another is not taken for it."""
    import torch

    tag = f"{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}.abi{int(torch._C._GLIBCXX_USE_CXX11_ABI)}"
    return os.path.join(LIB_DIR, f"s4d_decoder_calls.{tag.replace(os.sep, '_')}.so")


def build_calls(force: bool = False) -> str:
    """The Python module of csrc/decoder_calls.cpp (host code against torch's headers; it needs no nvcc)."""
    import torch
    from torch.utils.cpp_extension import include_paths

    src, path = os.path.join(CSRC, "decoder_calls.cpp"), calls_path()
    deps = [src, os.path.join(INCLUDE, "s4d_dfa.h"), os.path.join(INCLUDE, "s4d_decoder.h"), os.path.abspath(__file__)]
    if not force and os.path.exists(path) and all(os.path.getmtime(d) <= os.path.getmtime(path) for d in deps):
        return path
    os.makedirs(LIB_DIR, exist_ok=True)
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    dirs = [INCLUDE, *include_paths(), sysconfig.get_paths()["include"], cuda]
    _run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", *(a for d in dirs for a in ("-I", d)),
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-o", path + ".tmp", src, "-L",
          os.path.join(os.path.dirname(torch.__file__), "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"],
         "s4d_decoder_calls.so", False)
    os.replace(path + ".tmp", path)
    return path


def build(verbose_ptxas: bool = False, force: bool = False) -> str:
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    deps = srcs + [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith(".cuh")]
    deps.append(os.path.join(INCLUDE, "s4d_dfa.h"))
    if not force and os.path.exists(LIB_PATH):
        mt = os.path.getmtime(LIB_PATH)
        if all(os.path.getmtime(d) <= mt for d in deps) and not verbose_ptxas:
            return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    cmd = [nvcc_path(), *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "--shared", "-Xcompiler", "-fPIC",
           "-Xcompiler", "-fvisibility=hidden", "-I", INCLUDE, "-I", CSRC, "-o", LIB_PATH + ".tmp", *srcs,
           "-lcudart"]
    if verbose_ptxas:
        cmd[1:1] = ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libs4d_dfa.so")
    if verbose_ptxas:
        sys.stdout.write(res.stderr)
    os.replace(LIB_PATH + ".tmp", LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose-ptxas", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(a.verbose_ptxas, a.force))
    print(build_decoder(a.verbose_ptxas, a.force))
