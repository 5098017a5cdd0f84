"""Compile the CUDA library and the host module in-tree for sm_100a:  python -m medvision_b200.build

libmvr.so    the kernels behind the C ABI (nvcc; no torch)
_native.so   the Python package's host path on torch tensors (g++; links libmvr.so and torch)
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmvr.so")
NATIVE = os.path.join(HERE, "_native.so")
SOURCES = ["mvr_api.cu", "mvr_heads.cu", "mvr_window.cu", "mvr_encoder.cu"]  # one object file each
HEADERS = ["mvr_arith.cuh", "mvr_geom.cuh", "mvr_generic.cuh", "mvr_stream3d.cuh", "mvr_tma3d.cuh", "mvr_brick3d.cuh", "mvr_bwd3d.cuh", "mvr_offset.cuh", "mvr_cubic3d.cuh", "mvr_flat.cuh", "mvr_label.cuh", "mvr_plane2d.cuh", "mvr_elastic.cuh", "mvr_head.cuh",
           os.path.join("..", "..", "include", "mvr.h")]
ATTENTION_HEADERS = ["mvr_types.cuh", "mvr_span.cuh", "mvr_attn.cuh", "mvr_attn_fma.cuh", "mvr_attn_tc.cuh", "mvr_attn_tc_bwd.cuh", "mvr_attn_host.cuh", "mvr_tc.cuh",
                     os.path.join("..", "..", "include", "mvr.h")]
HEADERS_OF = {"mvr_api.cu": HEADERS, "mvr_heads.cu": ATTENTION_HEADERS + ["mvr_dropout.cuh", "mvr_logprob.cuh"], "mvr_window.cu": ATTENTION_HEADERS + ["mvr_attn_rows.cuh"],
              "mvr_encoder.cu": ["mvr_types.cuh", "mvr_norm.cuh", "mvr_rotary.cuh", os.path.join("..", "..", "include", "mvr.h")]}
LIB_FILES = sorted(set(SOURCES).union(*HEADERS_OF.values()))
NATIVE_SOURCES = ["mvr_torch.cpp", "mvr_torch_heads.cpp", "mvr_torch_encoder.cpp"]
NATIVE_HEADERS = ["mvr_torch.h", "mvr_torch_operators.h", os.path.join("..", "..", "include", "mvr.h")]

NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC"]
CXX_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-ffp-contract=off", "-w"]


def _older(target, files):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(os.path.join(CSRC, f)) > t for f in files)


def needs_build():
    return _older(LIB, LIB_FILES) or _older(NATIVE, NATIVE_SOURCES + NATIVE_HEADERS)


def _build_native():
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    includes = cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"]]
    # the system compiler and its shared libstdc++: a second, static copy of the C++ runtime in the module crashes in iostreams
    cmd = ["g++"] + CXX_FLAGS + ["-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI]
    for i in includes:
        cmd += ["-isystem", i]
    cmd += ["-o", NATIVE] + [os.path.join(CSRC, s) for s in NATIVE_SOURCES]
    for p in cpp_extension.library_paths("cuda"):
        cmd += ["-L" + p]
    cmd += ["-L" + HERE, "-Wl,-rpath,$ORIGIN", "-l:libmvr.so", "-ltorch_python", "-ltorch", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10",
            "-lcudart"]
    subprocess.check_call(cmd)


def build(force=False, verbose=False):
    """nvcc cross-compiles without a GPU; both .so stay beside the package."""
    if force or _older(LIB, LIB_FILES):
        nvcc = os.environ.get("NVCC", "nvcc")
        objects, running = [], []
        for source in SOURCES:
            objects.append(os.path.join(CSRC, os.path.splitext(source)[0] + ".o"))
            if force or _older(objects[-1], [source] + HEADERS_OF[source]):
                cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + \
                      ["-c", "-o", objects[-1], os.path.join(CSRC, source)]
                running.append((cmd, subprocess.Popen(cmd)))
        for cmd, process in running:
            if process.wait() != 0:
                raise subprocess.CalledProcessError(process.returncode, cmd)
        subprocess.check_call([nvcc] + NVCC_FLAGS + ["-shared", "-o", LIB] + objects)
    if force or _older(NATIVE, NATIVE_SOURCES + NATIVE_HEADERS):
        _build_native()
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
