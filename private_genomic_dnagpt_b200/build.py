"""Builds the engine's shared library in-tree with nvcc for sm_100a.

``python -m private_genomic_dnagpt_b200.build`` (or ``build()``) compiles every
``csrc/*.cu`` translation unit in parallel and links
``private_genomic_dnagpt_b200/libckks_b200.so``, and compiles
``csrc/torch_draft.cpp`` against the installed torch into
``private_genomic_dnagpt_b200/_draft.so`` (the drafted-decoding operators on
torch tensors).  Only stale objects are rebuilt.
"""

from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libckks_b200.so")
BINDING = os.path.join(HERE, "_draft.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
         "-Xcompiler", "-fPIC,-ffp-contract=off,-O2",
         "-Xptxas", "-O3"]


def _nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else (shutil.which("nvcc") or "nvcc")


def _host_compiler() -> list[str]:
    # the system g++ (an environment CC/CXX may point at a toolchain nvcc rejects)
    for c in ("/usr/bin/g++", shutil.which("g++")):
        if c and os.path.exists(c):
            return ["-ccbin", c]
    return []


def _deps_newer(obj: str, src: str) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    srcs = [src] + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.hpp")) + \
        glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    return any(os.path.getmtime(s) > t for s in srcs)


def _make(cmd: list[str], out: str, what: str) -> str:
    """Runs the compiler or linker; `out` appears whole or not at all, so that
    processes started together do not load what another has half written.
    Returns what it printed."""
    root, ext = os.path.splitext(out)
    part = f"{root}.{os.getpid()}{ext}"
    try:
        r = subprocess.run([*cmd, "-o", part], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{what}:\n{r.stdout}\n{r.stderr}")
        os.replace(part, out)
    finally:
        if os.path.exists(part):
            os.remove(part)
    return r.stderr


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ, os.path.basename(src).replace(".cu", ".o"))
    if _deps_newer(obj, src):
        cmd = [_nvcc(), *_host_compiler(), *ARCH, *FLAGS, "-c", src]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        printed = _make(cmd, obj, f"nvcc failed for {src}")
        if verbose:
            sys.stderr.write(printed)
    return obj


def build_binding() -> str:
    """The torch binding; needs the engine's library and torch."""
    src = os.path.join(CSRC, "torch_draft.cpp")
    deps = [src, os.path.join(HERE, "..", "include", "ckks_b200.h")]
    if os.path.exists(BINDING) and all(os.path.getmtime(d) <= os.path.getmtime(BINDING) for d in deps):
        return BINDING
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    gxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else (shutil.which("g++") or "g++")
    include = [f"-I{p}" for p in (*cpp_extension.include_paths(), sysconfig.get_path("include"),
                                  os.path.join(cuda, "include"))]
    cmd = [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", *include, "-DTORCH_EXTENSION_NAME=_draft",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", src, f"-L{libs}",
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", f"-L{HERE}",
           "-l:libckks_b200.so", f"-Wl,-rpath,{libs}",
           "-Wl,-rpath,$ORIGIN"]
    _make(cmd, BINDING, f"g++ failed for {src}")
    return BINDING


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        _make([_nvcc(), *_host_compiler(), *ARCH, "-shared", *objs, "-lcudart"], LIB, "link failed")
    try:
        import torch  # noqa: F401
    except ImportError:
        return LIB  # the engine itself needs no torch
    build_binding()
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
