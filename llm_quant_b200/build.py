"""Build liblq_sm100.so in-tree with nvcc for sm_100a (B200), and lq_torch.so, the
torch bindings in C++ of the calls whose host time counts, with the host compiler.

    python -m llm_quant_b200.build        # or: python llm_quant_b200/build.py

Each .cu under csrc/ is compiled to an object (in parallel, skipped when up
to date) and linked into llm_quant_b200/_lib/liblq_sm100.so.  The elementwise
quantization sources are compiled with --fmad=false on top of the explicit
__f*_rn intrinsics: the reference rounds after every torch op, so no two ops
may be contracted into one FMA.
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "_lib")
OBJDIR = os.path.join(HERE, "_lib", "obj")
LIB = os.path.join(LIBDIR, "liblq_sm100.so")
EXT = os.path.join(LIBDIR, "lq_torch.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-I", INCLUDE,
          "--expt-relaxed-constexpr"]
# sources whose arithmetic must not be contracted (bit-exact parity)
EXACT = {"lq_group.cu", "lq_kv.cu", "lq_nf4.cu", "lq_hadamard.cu", "lq_affine.cu", "lq_api.cu",
         "lq_kv4_store.cu"}


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers_mtime() -> float:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(OBJDIR, src.replace(".cu", ".o"))
    srcp = os.path.join(CSRC, src)
    if not force and os.path.exists(obj):
        if os.path.getmtime(obj) >= max(os.path.getmtime(srcp), _headers_mtime()):
            return obj
    flags = list(COMMON)
    if src in EXACT:
        flags += ["--fmad=false"]
    cmd = [nvcc()] + ARCH + flags + ["-c", srcp, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if verbose:
        sys.stderr.write(r.stderr)
    return obj


def _cxx() -> str:
    return os.environ.get("CXX") or "g++"


def _compile_ext(force: bool) -> str:
    """lq_torch.cpp against the installed torch's headers; again for another torch, Python or compiler."""
    import sysconfig
    import torch
    src, obj, made = os.path.join(CSRC, "lq_torch.cpp"), os.path.join(OBJDIR, "lq_torch.o"), os.path.join(OBJDIR, "lq_torch.for")
    key = f"torch {torch.__version__} python {sys.version} {_cxx()}"
    if not force and os.path.exists(obj) and os.path.exists(made):
        with open(made) as f:
            same = f.read() == key
        if same and os.path.getmtime(obj) >= max(os.path.getmtime(src), os.path.getmtime(os.path.join(INCLUDE, "lq_sm100.h"))):
            return obj
    root = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    cmd = [_cxx(), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-c", src, "-o", obj,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-DTORCH_API_INCLUDE_EXTENSION_H"]
    for d in (root, os.path.join(root, "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"]):
        cmd += ["-isystem", d]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"the host compiler failed for lq_torch.cpp:\n{r.stdout}\n{r.stderr}")
    with open(made, "w") as f:
        f.write(key)
    return obj


def _link_ext(obj: str, force: bool) -> None:
    if not force and os.path.exists(EXT) and os.path.getmtime(EXT) >= os.path.getmtime(obj):
        return
    import torch
    tmp = EXT + ".tmp"
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    # torch's own libstdc++, never a static one: two copies in a process do not share
    # their locales, and formatting a number in the second one ends it
    cmd = [_cxx(), "-shared", "-o", tmp, obj, LIB, "-Wl,-rpath,$ORIGIN", f"-L{libs}", "-lc10", "-ltorch_cpu", "-ltorch_python",
           "-lc10_cuda", "-ltorch_cuda", "-nodefaultlibs", "-l:libstdc++.so.6", "-lm", "-lgcc_s", "-lgcc", "-lc"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, EXT)


def build(force: bool = False, verbose: bool = False) -> str:
    """The library, which needs nvcc alone, and then the bindings, which need torch and a host compiler."""
    os.makedirs(OBJDIR, exist_ok=True)
    srcs = _sources()
    torch_there = importlib.util.find_spec("torch") is not None
    with ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        ext = ex.submit(_compile_ext, force) if torch_there else None
        objs = list(ex.map(lambda s: _compile(s, force, verbose), srcs))
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc()] + ARCH + ["-shared", "-Xlinker", "-soname=liblq_sm100.so", "-o", tmp] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    if ext is None:
        sys.stderr.write("no torch here: lq_torch.so, its bindings, is not built\n")
    else:
        _link_ext(ext.result(), force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
