"""Build ``libvoyager_b200.so`` in-tree with nvcc for sm_100a.

Every ``csrc/*.cu`` and ``csrc/*.cpp`` file is compiled to an object under
``_build/`` (in parallel, skipped when up to date) and linked into
``voyager_b200/libvoyager_b200.so``.  The CUDA runtime is linked statically,
so the library needs only the driver at run time.  No fast-math: the
numerics rely on IEEE division and round-to-nearest-even.

``csrc/py/vq_decode_py.cpp`` becomes ``voyager_b200/_decode.so``, the CPython
binding of the cached-decoding operators (g++, torch's headers and libraries).
"""

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
PROJ = os.path.dirname(PKG)
ROOT = os.path.dirname(PROJ)
CSRC = os.path.join(PROJ, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(ROOT, "_build")
OUT = os.path.join(PKG, "libvoyager_b200.so")
PY_SRC = os.path.join(CSRC, "py", "vq_decode_py.cpp")
PY_OUT = os.path.join(PKG, "_decode.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-ffp-contract=off",
          f"-I{INCLUDE}", f"-I{CSRC}"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _sources():
    out = []
    for f in sorted(os.listdir(CSRC)):
        if f.endswith((".cu", ".cpp")):
            out.append(os.path.join(CSRC, f))
    return out


def _headers_mtime():
    ts = [os.path.getmtime(os.path.join(INCLUDE, f)) for f in os.listdir(INCLUDE)]
    ts += [os.path.getmtime(os.path.join(CSRC, f)) for f in os.listdir(CSRC)
           if f.endswith((".cuh", ".h", ".hpp", ".inc"))]
    return max(ts) if ts else 0.0


def _compile(src: str, verbose: bool, extra) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if (os.path.exists(obj) and os.path.getmtime(obj) >= os.path.getmtime(src)
            and os.path.getmtime(obj) >= _headers_mtime()):
        return obj
    cmd = [nvcc(), *ARCH, *COMMON, *extra, "-c", src, "-o", obj]
    if src.endswith(".cpp"):
        cmd[1:1] = ["-x", "c++"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    if verbose and r.stderr.strip():
        print(r.stderr, file=sys.stderr)
    return obj


def _build_binding(verbose: bool) -> None:
    """``_decode.so``, linked with the library beside it and with torch's.  It
    holds torch's inline code and Python's ABI, so it is built again when the
    record of what it was built with (``_build/_decode.stamp``) differs."""
    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    inc = [os.path.join(root, "include"), os.path.join(root, "include/torch/csrc/api/include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-I{INCLUDE}", *[a for i in inc for a in ("-isystem", i)],
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", PY_SRC, "-o", PY_OUT + ".tmp",
           f"-L{PKG}", "-l:" + os.path.basename(OUT), f"-L{os.path.join(root, 'lib')}", "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    stamp = os.path.join(BUILD, "_decode.stamp")
    made_with = "\n".join([torch.__version__, str(sysconfig.get_config_var("SOABI")), " ".join(cmd)])
    newest = max(os.path.getmtime(f) for f in (PY_SRC, os.path.join(INCLUDE, "voyager_b200.h")))
    if os.path.exists(PY_OUT) and os.path.getmtime(PY_OUT) >= newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == made_with:
                return
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {PY_SRC}:\n{r.stdout}\n{r.stderr}")
    os.replace(PY_OUT + ".tmp", PY_OUT)
    with open(stamp, "w") as f:
        f.write(made_with)


def build(verbose: bool = False, extra=()) -> str:
    """Compile and link; returns the path of the shared object."""
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max(1, min(len(srcs), os.cpu_count() or 4))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose, list(extra)), srcs))
    newest = max(os.path.getmtime(o) for o in objs)
    if os.path.exists(OUT) and os.path.getmtime(OUT) >= newest:
        _build_binding(verbose)
        return OUT
    cmd = [nvcc(), *ARCH, "-shared", "-o", OUT + ".tmp", *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(OUT + ".tmp", OUT)
    _build_binding(verbose)
    return OUT


if __name__ == "__main__":
    print(build(verbose=True))
