"""Builds pdefa_b200/lib/libpdefa_native.so from pdefa_b200/csrc with nvcc.

The library is built in-tree (objects under pdefa_b200/_build, the shared object
under pdefa_b200/lib) for sm_100a only. Only the C-ABI entry points are exported
(-fvisibility=hidden + explicit default visibility on the API declarations).

Where a torch with CUDA is installed, lib/lm_torch-<python>-<torch>.so (pdefa_b200/torch_ext)
is built too: the binding of the language-model operators for torch tensors. It fits these
versions only, so they are part of its name. The engine does without it:
if it cannot be built, build() warns, and the first call of such an operator says why.

Usage: python -m pdefa_b200.build [--force] [--jobs N]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libpdefa_native.so")
TORCH_SRC = os.path.join(HERE, "torch_ext", "lm_torch.cpp")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(f for f in os.listdir(SRC) if f.endswith((".cu", ".cpp")))


def _newest_header() -> float:
    hs = [os.path.join(SRC, f) for f in os.listdir(SRC) if f.endswith((".h", ".cuh"))]
    inc = os.path.join(os.path.dirname(HERE), "include")
    hs += [os.path.join(inc, f) for f in os.listdir(inc)]
    return max(os.path.getmtime(h) for h in hs)


def compile_one(src: str, force: bool) -> str:
    obj = os.path.join(BUILD, src + ".o")
    path = os.path.join(SRC, src)
    if (not force and os.path.exists(obj) and os.path.getmtime(obj) >= os.path.getmtime(path)
            and os.path.getmtime(obj) >= _newest_header()):
        return obj
    cmd = [nvcc(), "-std=c++17", "-O3", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC",
           "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr", "-c", path, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def torch_root():
    """The installed torch's folder; None without torch or where it has no CUDA."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:
        return None
    root = os.path.dirname(spec.origin)
    return root if os.path.exists(os.path.join(root, "lib", "libc10_cuda.so")) else None


def torch_lib(root: str) -> str:
    """The binding for this Python and the torch at `root`, whose version is read without importing it."""
    with open(os.path.join(root, "version.py")) as f:
        found = re.search(r"^__version__\s*=\s*['\"]([\w.+-]+)['\"]", f.read(), re.M)
    if not found:
        raise RuntimeError(f"torch binding: no version in {f.name}")
    return os.path.join(LIB_DIR, f"lm_torch-{sys.implementation.cache_tag}-{found.group(1)}.so")


def build_torch_binding(force: bool) -> None:
    """Builds torch_lib() unless it is up to date or there is no torch with CUDA to bind. Raises
    RuntimeError with the compiler's output."""
    root = torch_root()
    if root is None:
        return
    lib = torch_lib(root)
    if (not force and os.path.exists(lib)
            and os.path.getmtime(lib) >= max(os.path.getmtime(TORCH_SRC), _newest_header())):
        return
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], cuda]
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", *("-I" + i for i in inc), TORCH_SRC,
           "-o", lib + ".tmp", "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_python"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"torch binding: {e}") from e
    if r.returncode != 0:
        raise RuntimeError(f"torch binding failed:\n{r.stdout}\n{r.stderr}")
    os.replace(lib + ".tmp", lib)


def build(force: bool = False, jobs: int = 0) -> str:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs) + 1, os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(jobs) as ex:
        binding = ex.submit(build_torch_binding, force)
        objs = list(ex.map(lambda s: compile_one(s, force), srcs))
    if (force or not os.path.exists(LIB)
            or max(os.path.getmtime(o) for o in objs) > os.path.getmtime(LIB)):
        cmd = [nvcc(), "-shared", *ARCH, "-cudart", "static", "-o", LIB + ".tmp", *objs, "-lpthread", "-ldl", "-lrt", "-lz"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(LIB + ".tmp", LIB)
    try:
        binding.result()
    except RuntimeError as e:
        warnings.warn(f"the language-model operators have no binding for torch tensors: {e}", RuntimeWarning, stacklevel=2)
    return LIB


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=0)
    a = ap.parse_args(argv)
    print(build(a.force, a.jobs))


if __name__ == "__main__":
    sys.exit(main())
