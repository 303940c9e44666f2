"""Build liboasr_b200.so in-tree (openasr_b200/liboasr_b200.so) with nvcc for
sm_100a only.  Usage: python -m openasr_b200.build  (or build() from Python)."""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "liboasr_b200.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")  # the Python binding's short way (csrc/torch_ops.cc)
ROOT = os.path.dirname(HERE)

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc")
# The image exports CXX=/opt/gcc/bin/g++; the system g++ on PATH is used as host compiler.
HOST_CXX = shutil.which("g++", path="/usr/bin") or "g++"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
    "-Xcompiler", "-ffp-contract=off", "-ccbin", HOST_CXX, "-I", os.path.join(ROOT, "include"),
]
CXX_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-ffp-contract=off", "-pthread", "-I", os.path.join(ROOT, "include")]


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu"))), sorted(glob.glob(os.path.join(CSRC, "*.cpp")))


def _headers_mtime() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + [
        os.path.join(ROOT, "include", "oasr_b200.h")]
    return max(os.path.getmtime(h) for h in hs)


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), _headers_mtime()):
        return obj
    if src.endswith(".cu"):
        cmd = [NVCC] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
    else:
        cmd = [HOST_CXX] + CXX_FLAGS + ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    if verbose and r.stderr:
        sys.stderr.write(r.stderr)
    return obj


def _build_torch_ops() -> None:
    """The Python binding's extension, for the torch that is installed.  Without torch's headers, or
    where they do not compile, there is none and the binding goes through ctypes (slower, the same calls)."""
    spec = importlib.util.find_spec("torch")
    torch = os.path.dirname(spec.origin) if spec and spec.origin else ""
    src, inc = os.path.join(CSRC, "torch_ops.cc"), sysconfig.get_path("include")
    stamp = TORCH_OPS + ".for"  # which torch and Python it was built for: another one's may not be loaded
    if not (os.path.exists(os.path.join(torch, "include", "torch", "csrc", "autograd", "python_variable.h"))
            and os.path.exists(os.path.join(inc, "Python.h"))):
        _remove(TORCH_OPS, stamp)
        return
    with open(os.path.join(torch, "version.py")) as f:
        wants = f"{sys.version}\n{torch}\n{f.read()}"
    if os.path.exists(TORCH_OPS) and os.path.getmtime(TORCH_OPS) >= max(os.path.getmtime(src), _headers_mtime()) and \
            os.path.exists(stamp) and open(stamp).read() == wants:
        return
    _remove(TORCH_OPS, stamp)
    cmd = [HOST_CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-I", os.path.join(ROOT, "include"), "-I", inc,
           "-isystem", os.path.join(torch, "include"), src, "-o", TORCH_OPS, "-L", os.path.join(torch, "lib"),
           "-ltorch_python", "-ltorch_cpu", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        _remove(TORCH_OPS)
        sys.stderr.write(f"the Python binding's extension does not compile, its calls go through ctypes: {' '.join(cmd)}\n{r.stderr}")
        return
    with open(stamp, "w") as f:
        f.write(wants)


def _remove(*paths: str) -> None:
    for p in paths:
        if os.path.exists(p):
            os.remove(p)


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    _build_torch_ops()
    cu, cpp = _sources()
    with cf.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), cu + cpp))
    if os.path.exists(LIB) and os.path.getmtime(LIB) >= max(os.path.getmtime(o) for o in objs):
        return LIB
    cmd = [NVCC] + ARCH + ["-shared", "-ccbin", HOST_CXX, "-o", LIB] + objs + ["-lpthread"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
