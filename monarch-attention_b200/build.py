"""Build libmonarch_attn.so in-tree with nvcc for sm_100a, and the key-value
cache's binding for torch tensors (_ma_torch.*.so) with the host compiler.

The library is a plain C-ABI shared object (include/ma_api.h): no torch
headers, cudart linked statically, the driver's cuTensorMapEncodeTiled
resolved at run time through cudaGetDriverEntryPoint.  The binding belongs to
one Python and one torch, which its name says; without it the library is
whole, and the key-value cache's Python calls raise.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT = os.path.join(HERE, "libmonarch_attn.so")
BINDING_SRC = os.path.join(CSRC, "ma_torch.cpp")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
              "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return (sources() + glob.glob(os.path.join(CSRC, "*.cuh"))
            + glob.glob(os.path.join(INCLUDE, "*.h")) + [os.path.abspath(__file__)])


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(d) <= t for d in _deps())


def binding_path() -> str:
    """Where the binding for this Python and this torch lies: one made for others
    must not be loaded."""
    import torch
    return os.path.join(HERE, f"_ma_torch.{sys.implementation.cache_tag}-torch-{torch.__version__}.so")


def binding_up_to_date() -> bool:
    out = binding_path()
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(d) <= t for d in
               (BINDING_SRC, os.path.join(INCLUDE, "ma_api.h"), os.path.abspath(__file__)))


def build_binding() -> str:
    """Compile csrc/ma_torch.cpp against this interpreter's torch.  One that was
    built from older sources is taken away first: it must not outlive a failure."""
    import sysconfig

    import torch
    out = binding_path()
    if os.path.exists(out):
        os.remove(out)
    root = os.path.join(os.path.dirname(os.path.abspath(torch.__file__)))
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    tmp = f"{out}.{os.getpid()}.tmp"
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(f"-I{d}" for d in (INCLUDE, os.path.join(root, "include"),
                                os.path.join(root, "include", "torch", "csrc", "api", "include"),
                                os.path.join(cuda, "include"), sysconfig.get_paths()["include"])),
           BINDING_SRC, "-o", tmp, f"-L{os.path.join(root, 'lib')}",
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {BINDING_SRC}:\n{res.stderr[-4000:]}")
    os.replace(tmp, out)
    return out


def build(force: bool = False, verbose: bool = False, out: str = OUT,
          defines: tuple = ()) -> str:
    """Compile every .cu under csrc/ (one nvcc per file, in parallel) and link
    libmonarch_attn.so; returns its path.  The in-tree build makes the torch
    binding after it; where that fails (no torch or host compiler here) it warns.

    ``defines`` adds -D flags (e.g. ("MA_TC_TRACE",) for the per-item timeline
    build, written to a separate ``out`` path).
    """
    if force or out != OUT or not up_to_date():
        build_library(verbose, out, defines)
    if out == OUT:
        try:
            if force or not binding_up_to_date():
                build_binding()
        except (ImportError, OSError, RuntimeError) as e:
            warnings.warn(f"the key-value cache's torch binding was not built: {e}")
    return out


def build_library(verbose: bool, out: str, defines: tuple) -> None:
    from concurrent.futures import ThreadPoolExecutor
    import tempfile
    objdir = tempfile.mkdtemp(prefix="ma_build_")
    dflags = [f"-D{d}" for d in defines]
    compile_flags = [f for f in NVCC_FLAGS if f != "-shared"]

    def compile_one(src):
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc(), *ARCH_FLAGS, *compile_flags, *dflags, "-I", INCLUDE, "-c", "-o", obj, src]
        return obj, cmd, subprocess.run(cmd, capture_output=True, text=True)

    srcs = sources()
    with ThreadPoolExecutor(max_workers=min(len(srcs), os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, srcs))
    log = os.path.join(HERE, "build.log")
    tmp = out + ".tmp"
    link = [nvcc(), *ARCH_FLAGS, "-shared", "-o", tmp, *[r[0] for r in results]]
    with open(log, "w") as f:
        for obj, cmd, res in results:
            f.write(" ".join(cmd) + "\n" + res.stdout + res.stderr)
        bad = [r for r in results if r[2].returncode != 0]
        if bad:
            shutil.rmtree(objdir, ignore_errors=True)
            raise RuntimeError(f"nvcc failed (see {log}):\n" +
                               "\n".join(r[2].stderr[-4000:] for r in bad))
        res = subprocess.run(link, capture_output=True, text=True)
        f.write(" ".join(link) + "\n" + res.stdout + res.stderr)
    shutil.rmtree(objdir, ignore_errors=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed (see {log}):\n{res.stderr[-4000:]}")
    if verbose:
        print(open(log).read())
    os.replace(tmp, out)


if __name__ == "__main__":
    print(build(force=True, verbose=True))
