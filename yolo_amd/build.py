"""Builds yolo_amd/libyolo_amd.so from yolo_amd/csrc/*.hip with hipcc for gfx950, and yolo_amd/_torch_ops.so, the torch
binding of the token operators, from csrc/yamd_torch.cpp with the host compiler.

The library is built in-tree so the same file is what tests, bench.py and smoke() load; there is
no JIT and no fallback: if the .so is missing, ``yolo_amd.lib`` raises.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "_obj")
LIB = os.path.join(HERE, "libyolo_amd.so")

# (source, extra flags).  decode/nms follow the reference's fp32 operation order exactly, so the
# compiler must not fuse a*b+c into an fma there.
SOURCES = [
    ("yamd_core.hip", []),
    ("yamd_conv.hip", []),
    ("yamd_conv_k1.hip", []),
    ("yamd_conv_k1b.hip", []),
    ("yamd_conv_k3s1.hip", []),
    ("yamd_conv_k3s1b.hip", []),
    ("yamd_conv_k3s2.hip", []),
    ("yamd_conv_k3s2b.hip", []),
    ("yamd_decode.hip", ["-ffp-contract=off"]),
    ("yamd_nms.hip", ["-ffp-contract=off"]),
    ("yamd_preprocess.hip", ["-ffp-contract=off"]),
    ("yamd_metric.hip", ["-ffp-contract=off"]),
    ("yamd_stem.hip", []),
    ("yamd_bneck.hip", []),
    ("yamd_c3.hip", []),
    ("yamd_microbench.hip", []),
    ("yamd_layer_norm.hip", []),
    ("yamd_attention.hip", []),
    ("yamd_attention_backward.hip", []),
    ("yamd_relative_bias.hip", []),
    ("yamd_plan.hip", []),
]
# (no packed float32 instructions: the feature is switched off for the device; the host pass does not know it and says so)
COMMON = ["-O3", "-std=c++17", "-fPIC", "--offload-arch=gfx950", "-Wall", "-Wno-unused-function",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
HEADERS = [os.path.join(CSRC, "yamd_common.h"), os.path.join(CSRC, "yamd_conv_kernel.h"),
           os.path.join(CSRC, "yamd_conv_variants.inc"), os.path.join(CSRC, "yamd_attention.h"),
           os.path.join(CSRC, "yamd_distance.h"),
           os.path.join(HERE, "..", "include", "yolo_amd.h")]


BINDING_SRC = os.path.join(CSRC, "yamd_torch.cpp")
BINDING = os.path.join(HERE, "_torch_ops.so")


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "hipcc"


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build_library(force: bool = False, verbose: bool = True) -> str:
    os.makedirs(OBJ, exist_ok=True)
    hipcc = _hipcc()
    jobs = []
    objs = []
    for src, extra in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ, src.replace(".hip", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + HEADERS):
            jobs.append([hipcc] + COMMON + extra + ["-c", s, "-o", o])

    def run(cmd):
        if verbose:
            print("[yolo_amd.build]", " ".join(cmd), flush=True)
        subprocess.check_call(cmd)

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            list(ex.map(run, jobs))
    if force or jobs or _stale(LIB, objs):
        run([hipcc, "-shared", "-fPIC", "--offload-arch=gfx950", "-o", LIB] + objs)
    return LIB


def build_binding(force: bool = False, verbose: bool = True) -> str:
    """Host code over the C ABI and torch's C++ API; needs libyolo_amd.so to link against."""
    header = os.path.join(HERE, "..", "include", "yolo_amd.h")
    if not force and not _stale(BINDING, [BINDING_SRC, header]):
        return BINDING
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for inc in include_paths() + [os.path.join(rocm, "include"), sysconfig.get_paths()["include"]]:
        cmd += ["-isystem", inc]
    cmd += [BINDING_SRC, "-o", BINDING, "-L" + torch_lib, "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python",
            "-L" + HERE, "-l:libyolo_amd.so", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print("[yolo_amd.build]", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return BINDING


if __name__ == "__main__":
    build_library(force="--force" in sys.argv)
    build_binding(force="--force" in sys.argv)
    print(LIB)
