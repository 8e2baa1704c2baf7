"""Builds the HIP backend library in-tree.

  1. hipcc --genco for gfx950: each file of precompiled kernels -> a code object;
  2. the code objects are embedded into C files as byte arrays;
  3. hipcc -c: noalloc.hip (a device array and its address lookup);
  4. gcc (plain C, HIP runtime C API) -> tinyhvm_amd/libthvm_hip.so.

Run: python -m tinyhvm_amd.build
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INC = os.path.join(ROOT, "include")
BUILD = os.path.join(ROOT, "_build")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
LIB_NAME = "libthvm_hip.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)

# no FP contraction: a*b+c stays two rounded operations, as in the x86 engine
HIP_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
HOST_SOURCES = ["backend.c", "pool.c", "kgen.c", "rtc.c", "affine.c", "dense.c", "window.c", "chain.c", "block.c", "replay.c"]
KERNEL_SOURCES = ["static_kernels.hip", "norm_kernels.hip", "gemm_kernels.hip"]
# operators the engine has no counterpart of, whose roundings no one else repeats
CONTRACTED = {"norm_kernels.hip", "gemm_kernels.hip"}
# host + device code built by hipcc into an object: the static device workspace
# of the no-allocation entry point, whose address hipGetSymbolAddress looks up
HIP_OBJECTS = ["noalloc.hip"]


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        raise RuntimeError("build step failed: %s" % cmd[0])
    return r


def _embed(source):
    """C file that holds the code object of one kernel source as
    thvm_<name>_co."""
    name = os.path.splitext(source)[0]
    co = os.path.join(BUILD, name + ".hsaco")
    flags = ["-ffp-contract=fast" if f == "-ffp-contract=off" and source in CONTRACTED else f for f in HIP_FLAGS]
    _run([os.path.join(ROCM, "bin", "hipcc"), "--genco"] + flags +
         ["-I" + INC, "-I" + CSRC, os.path.join(CSRC, source), "-o", co])
    data = open(co, "rb").read()
    blob = os.path.join(BUILD, name + "_blob.c")
    with open(blob, "w") as f:
        f.write("/* generated by tinyhvm_amd/build.py from a kernel code object */\n")
        f.write("__attribute__((aligned(4096))) const unsigned char thvm_%s_co[%d] = {\n" % (name, len(data)))
        for i in range(0, len(data), 24):
            f.write("  " + ",".join(str(b) for b in data[i:i + 24]) + ",\n")
        f.write("};\n")
        f.write("const unsigned long thvm_%s_co_len = %dUL;\n" % (name, len(data)))
    return blob


def build_kernels():
    os.makedirs(BUILD, exist_ok=True)
    with ThreadPoolExecutor(len(KERNEL_SOURCES)) as pool:
        return list(pool.map(_embed, KERNEL_SOURCES))


def build_hip_objects():
    os.makedirs(BUILD, exist_ok=True)
    objs = []
    for s in HIP_OBJECTS:
        obj = os.path.join(BUILD, os.path.splitext(s)[0] + ".o")
        _run([os.path.join(ROCM, "bin", "hipcc"), "-c", "-fPIC"] + HIP_FLAGS +
             ["-I" + INC, "-I" + CSRC, os.path.join(CSRC, s), "-o", obj])
        objs.append(obj)
    return objs


def build_library():
    blobs = build_kernels()
    objs = build_hip_objects()
    srcs = [os.path.join(CSRC, s) for s in HOST_SOURCES if os.path.exists(os.path.join(CSRC, s))]
    tmp = LIB_PATH + ".tmp"
    _run(["gcc", "-std=gnu11", "-O2", "-fPIC", "-shared", "-Wall", "-Wno-unused-function",
          "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROCM, "include"), "-I" + INC, "-I" + CSRC]
         + srcs + blobs + objs + ["-L" + os.path.join(ROCM, "lib"), "-lamdhip64", "-lhiprtc",
                                   "-lstdc++", "-lpthread", "-lm", "-Wl,-rpath," + os.path.join(ROCM, "lib"),
                                   "-o", tmp])
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main():
    path = build_library()
    print("built", path)


if __name__ == "__main__":
    main()
