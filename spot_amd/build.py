"""Build libstes_hip.so (gfx950) in-tree with hipcc, and _stes_torch.so (host code on torch's C++ interface) on top of it.  No GPU needed."""
import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libstes_hip.so")
TORCH_SRC = os.path.join(CSRC, "stes_torch.cpp")
TORCH_LIB = os.path.join(HERE, "_stes_torch.so")
# No packed fp32 arithmetic (v_pk_add_f32, v_pk_mul_f32, v_pk_fma_f32; the compiler forms them by itself from ordinary float
# code): some of their forms have given wrong results on this card now and then.  The host pass does not know the feature and warns.
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _torch_command():
    torch = os.path.dirname(importlib.util.find_spec("torch").origin)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    inc = [f"{torch}/include", f"{torch}/include/torch/csrc/api/include", f"{rocm}/include", sysconfig.get_paths()["include"]]
    return (["g++", "-O2", "-fPIC", "-shared", "-std=c++17", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1"] + [f for i in inc for f in ("-isystem", i)]
            + [TORCH_SRC, "-o", TORCH_LIB, f"-L{torch}/lib", f"-L{HERE}", "-l:libstes_hip.so", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch",
               "-ltorch_python", "-Wl,-rpath,$ORIGIN"])


def _newer(lib, deps):
    return os.path.exists(lib) and all(os.path.getmtime(lib) >= os.path.getmtime(d) for d in deps)


def build(force=False, verbose=True):
    build_kernels(force, verbose)
    if force or not _newer(TORCH_LIB, [TORCH_SRC, os.path.join(HERE, "..", "include", "stes.h"), os.path.abspath(__file__)]):
        cmd = _torch_command()
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return LIB


def build_kernels(force=False, verbose=True):
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    deps = srcs + glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(HERE, "..", "include", "stes.h"), os.path.abspath(__file__)]
    if not force and _newer(LIB, deps):
        return LIB
    objs = []
    procs = []
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    for s in srcs:
        o = os.path.join(HERE, "build", os.path.basename(s) + ".o")
        objs.append(o)
        if not force and _newer(o, [s] + deps[len(srcs):]):
            continue
        cmd = ["hipcc"] + FLAGS + ["-c", s, "-o", o]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((s, subprocess.Popen(cmd)))
    for s, p in procs:
        if p.wait() != 0:
            raise RuntimeError(f"hipcc failed on {s}")
    cmd = ["hipcc", "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
