"""Build libsmoe_b200.so (sm_100a only) in-tree with nvcc.

    python supersonic-moe_b200/build.py [--force] [--verbose]

The library lands next to the Python package (sonicmoe/libsmoe_b200.so) and is
loaded with ctypes; it links nothing but the CUDA runtime.  Beside it lies
sonicmoe/_host.so, which calls it on torch tensors (csrc/host_torch.cpp): made
with the installed PyTorch, and again when that is another; without one it is
left out.
"""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT = os.path.join(HERE, "sonicmoe", "libsmoe_b200.so")
SOURCES = ["routing.cu", "quant.cu", "combine.cu", "glu.cu", "ep_plan.cu", "ep_peer.cu", "gemm.cu", "layer.cu",
           "group_routing.cu", "quant128.cu", "gemm128.cu", "block128.cu",
           "norm.cu", "grad_norm.cu", "grouped.cu"]
HOST_SOURCE = os.path.join(CSRC, "host_torch.cpp")
HOST_OUT = os.path.join(HERE, "sonicmoe", "_host.so")
HOST_MADE = os.path.join(HERE, "build", "_host.command")      # what it was made by
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-I", INCLUDE, "-I", CSRC]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def host_command():
    """What compiles _host.so with the PyTorch and the Python that run this; None without a PyTorch."""
    try:
        import torch
    except ImportError:
        return None
    at = os.path.dirname(torch.__file__)
    return ([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DSMOE_TORCH_VERSION="{torch.__version__}"']
            + [a for i in (INCLUDE, os.path.join(at, "include"), os.path.join(at, "include", "torch", "csrc", "api", "include"),
                           sysconfig.get_paths()["include"], "/usr/local/cuda/include") for a in ("-I", i)]
            + [HOST_SOURCE, "-o", HOST_OUT, "-L", os.path.dirname(OUT), "-lsmoe_b200", "-L", os.path.join(at, "lib"), "-ltorch_python",
               "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"])


def _made_by(command):
    return "\n".join([sys.version, *command]) + "\n"


def host_stale(command):
    """Older than what it is made of, or made by another command, PyTorch or Python."""
    if not os.path.exists(HOST_MADE) or _stale(HOST_OUT, [HOST_SOURCE, os.path.join(INCLUDE, "smoe_b200.h")]):
        return True
    with open(HOST_MADE) as f:
        return f.read() != _made_by(command)


def build(force=False, verbose=False):
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(os.path.join(INCLUDE, "smoe_b200.h"))
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    objs, procs = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + headers):
            cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o]
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            print(out)
        if p.returncode:
            raise RuntimeError(f"nvcc failed on {src}")
    if force or procs or _stale(OUT, objs):
        cmd = [nvcc, "-shared", "-o", OUT] + objs + ["-lcudart"]
        subprocess.check_call(cmd)
    command = host_command()
    if command is None:
        print("no PyTorch: _host.so, which the operators around the experts are called through, is not built")
    elif force or host_stale(command):
        if os.path.exists(HOST_MADE):
            os.remove(HOST_MADE)
        subprocess.check_call(command)
        with open(HOST_MADE, "w") as f:
            f.write(_made_by(command))
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
