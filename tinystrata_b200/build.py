"""Build libtsb_moe.so in-tree for sm_100a (nvcc), after generating the GGUF codebook header.

``python -m tinystrata_b200.build`` or ``tinystrata_b200.build.build()``.  The library lands next to this file so it
travels with the source tree; nothing is installed into site-packages.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtsb_moe.so")
EXT = os.path.join(HERE, "_serving.so")          # the CPython module over the library (tinystrata_b200/serving.py)
EXT_FOR = os.path.join(HERE, "_build", "_serving.torch")   # the torch that it was built against
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
SOURCES = ["tsb_moe.cu", "tsb_decode.cu", "tsb_decode_act.cu", "tsb_ep.cu", "tsb_staged.cu", "tsb_cache.cu",
           "tsb_delta.cu", "tsb_gguf.cpp"]
# every header of the sources: a change to any of them rebuilds both objects
HEADERS = sorted(f for f in os.listdir(CSRC) if f.endswith((".cuh", ".inc"))) + ["../../include/tsb_moe.h"]
FLAGS = ["-std=c++17", "-O3", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-Xcompiler", "-fPIC",
         "--expt-relaxed-constexpr"]


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, force: bool = False) -> str:
    sys.path.insert(0, CSRC)
    try:
        import gen_codebooks
        gen_codebooks.main(os.path.join(CSRC, "codebooks.inc"))
    finally:
        sys.path.pop(0)
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    deps = [os.path.join(CSRC, f) for f in srcs + HEADERS]
    objs = []
    os.makedirs(os.path.join(HERE, "_build"), exist_ok=True)
    procs = []
    for s in srcs:
        obj = os.path.join(HERE, "_build", os.path.splitext(s)[0] + ".o")
        objs.append(obj)
        if force or _stale(obj, deps):
            cmd = [NVCC, *FLAGS, "-c", os.path.join(CSRC, s), "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((s, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for s, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {s}:\n{out}")
        if verbose and out.strip():
            print(out)
    if force or _stale(LIB, objs):
        cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB, *objs, "-lcudart", "-ldl"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    build_ext(verbose, force)
    return LIB


def build_ext(verbose: bool = False, force: bool = False) -> str:
    """The native Python module of the serving-step operators: C++ against torch's headers and the library beside it."""
    import sysconfig

    import torch

    src = os.path.join(CSRC, "tsb_pyserving.cpp")
    abi = int(torch.compiled_with_cxx11_abi())
    tag, known = f"torch {torch.__version__}, C++11 ABI {abi}\n", ""
    if os.path.exists(EXT_FOR):
        with open(EXT_FOR) as f:
            known = f.read()
    if not (force or known != tag or _stale(EXT, [src, os.path.join(HERE, "..", "include", "tsb_moe.h")])):
        return EXT
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(NVCC), "..", "include")]
    libs = os.path.join(root, "lib")
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *[f"-I{i}" for i in inc], src, "-o", EXT,
           f"-L{HERE}", "-l:libtsb_moe.so", f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on tsb_pyserving.cpp:\n{r.stderr}")
    os.makedirs(os.path.dirname(EXT_FOR), exist_ok=True)
    with open(EXT_FOR, "w") as f:
        f.write(tag)
    return EXT


if __name__ == "__main__":
    print(build(verbose=True, force="--force" in sys.argv))
