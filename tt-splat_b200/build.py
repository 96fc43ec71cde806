"""Build ``libttsplat_b200.so`` (sm_100a) and the torch functions over it in-tree, with nvcc and g++.

Each ``csrc/*.cu`` compiles to an object with relocatable device code (the device status word
is shared across translation units), then nvcc links them into one shared library next to this
file: ``build_library``, which needs neither torch nor Python's headers.  ``csrc/torch_ops.cpp`` (torch
functions over the C entry points) compiles with g++ against the installed torch into
``_torch_ops.so``, which links to that library: ``build_torch_ops``.  Objects are rebuilt only when a
source or header is newer.  Usage (without torch it builds the library alone):

    python tt-splat_b200/build.py            # or __graft_entry__.build()
"""
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libttsplat_b200.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-rdc=true", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
         "--expt-relaxed-constexpr", "-I", INCLUDE]


def nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA library cannot be built")


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers_mtime():
    paths = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    paths += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max((os.path.getmtime(p) for p in paths), default=0.0)


def _torch_ops_command():
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    gxx = os.environ.get("CXX") or shutil.which("g++")
    if not gxx:
        raise RuntimeError("g++ not found: the torch functions cannot be built")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    inc = cpp_extension.include_paths() + [cuda, sysconfig.get_paths()["include"]]
    lib = cpp_extension.library_paths()
    return [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_torch_ops",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in inc),
            # the C++ library before torch's, which carry parts of another one
            os.path.join(CSRC, "torch_ops.cpp"), "-o", TORCH_OPS, "-Wl,--no-as-needed", "-l:libstdc++.so.6",
            *(f"-L{p}" for p in lib), f"-L{HERE}", "-lttsplat_b200", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]


def _torch_ops_key(cmd):
    """What the extension is built against, beside its sources: the command (paths, C++ ABI), torch and
    Python."""
    import torch
    return "\n".join([torch.__version__, sys.version, *cmd])


def build_torch_ops(verbose=True):
    """``_torch_ops.so``; needs the CUDA library to link to.  Rebuilt when a source or header is newer, or when
    torch, Python or the command are others than it was built with."""
    src = os.path.join(CSRC, "torch_ops.cpp")
    newest = max(os.path.getmtime(src), _headers_mtime())
    cmd = _torch_ops_command()
    key, stamp = _torch_ops_key(cmd), os.path.join(BUILD, "torch_ops.stamp")
    built = None
    if os.path.exists(TORCH_OPS) and os.path.exists(stamp):
        with open(stamp) as f:
            built = f.read()
    if built != key or os.path.getmtime(TORCH_OPS) < newest:
        if verbose:
            print("torch_ops.cpp -o _torch_ops.so", flush=True)
        os.makedirs(BUILD, exist_ok=True)
        # under another name first: a build that fails or is cut off leaves what was there
        part = os.path.splitext(TORCH_OPS)[0] + ".part.so"
        cmd[cmd.index("-o") + 1] = part
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("g++ failed on torch_ops.cpp")
        os.replace(part, TORCH_OPS)
        with open(stamp, "w") as f:
            f.write(key)
    return TORCH_OPS


def build_library(verbose=True, extra_flags=()):
    os.makedirs(BUILD, exist_ok=True)
    cc = nvcc()
    hdr = _headers_mtime()
    jobs = []
    objs = []
    for src in _sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src[:-3] + ".o")
        objs.append(o)
        if not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr):
            jobs.append([cc, *ARCH, *FLAGS, *extra_flags, "-c", s, "-o", o])
    with cf.ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1)) as ex:
        for cmd, res in zip(jobs, ex.map(lambda c: subprocess.run(c, capture_output=True, text=True), jobs)):
            if verbose:
                print(" ".join(os.path.basename(x) if x.endswith((".cu", ".o")) else x for x in cmd[-3:]), flush=True)
            if res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
                raise RuntimeError(f"nvcc failed on {cmd[-3]}")
            if res.stderr.strip() and verbose:
                sys.stderr.write(res.stderr)
    if jobs or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        cmd = [cc, *ARCH, "-shared", "-o", LIB, *objs]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("nvcc link failed")
    return LIB


def build_all(verbose=True):
    """The CUDA library, and the torch functions where torch is installed."""
    build_library(verbose)
    if importlib.util.find_spec("torch") is not None:
        build_torch_ops(verbose)
    elif verbose:
        print("torch is not installed: built the CUDA library without the torch functions", flush=True)
    return LIB


if __name__ == "__main__":
    print(build_all())
