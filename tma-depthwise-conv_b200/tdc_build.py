"""Build the in-tree binaries of the package (run from anywhere):

  libtdc_sm100.so                 nvcc, -gencode arch=compute_100a,code=sm_100a:
                                  the kernels + the C ABI of include/tdc_dwconv.h
                                  and include/tdc_sequence.h, one object a source
                                  (static cudart, no libcuda link: the TMA encoder
                                  is fetched with cudaGetDriverEntryPoint)
  _tma_dwconv_C<EXT_SUFFIX>       g++: the PyTorch extension (csrc/bindings*.cpp),
                                  linked to libtdc_sm100.so through rpath $ORIGIN

Both land next to this file, so the directory is importable as-is
(``import tma_dwconv`` with this directory on ``sys.path``).  Rebuilds only
what is older than its sources.
"""
from __future__ import annotations

import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB = os.path.join(HERE, "libtdc_sm100.so")
EXT = os.path.join(HERE, "_tma_dwconv_C" + sysconfig.get_config_var("EXT_SUFFIX"))

# (No --split-compile: it builds ~4x faster but, with every instantiation in
# one translation unit, made the 7x7 direct-scheme kernels spill ~800 B.)
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC,-fvisibility=hidden", "-Xptxas", "-v"]


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd: list[str]) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout[-6000:] + r.stderr[-6000:])
        raise RuntimeError(f"build step failed: {cmd[0]}")
    return r.stdout + r.stderr


#: The library's translation units.
UNITS = ("tdc_capi.cu", "tdc_sequence.cu")
EXT_SOURCES = ("bindings.cpp", "bindings_sequence.cpp")


def _deps(*names: str) -> list[str]:
    """The sources `names` and every file of this repository that they include,
    directly or through one another."""
    found, todo = {}, list(names)
    while todo:
        name = todo.pop()
        if name in found:
            continue
        found[name] = next(p for p in (os.path.join(d, name) for d in (CSRC, INCLUDE))
                           if os.path.exists(p))
        with open(found[name]) as f:
            todo += re.findall(r'^[ \t]*#[ \t]*include[ \t]*"([^"]+)"', f.read(), re.M)
    return sorted(found.values())


def _tmp(path: str) -> str:
    """A temporary name beside `path`: a binary is written there and renamed
    into place, so no reader ever sees a partly written file."""
    d, f = os.path.split(path)
    return os.path.join(d, f".{f}.{os.getpid()}.tmp")


def _build_unit(nvcc: str, name: str, force: bool) -> str:
    """Object file of one .cu source, with its ptxas report beside it."""
    obj = os.path.join(HERE, name.replace(".cu", ".o"))
    if force or _stale(obj, _deps(name)):
        tmp = _tmp(obj)
        out = _run([nvcc, *NVCC_FLAGS, "-c", f"-I{INCLUDE}", f"-I{CSRC}",
                    os.path.join(CSRC, name), "-o", tmp])
        os.replace(tmp, obj)
        with open(obj.replace(".o", ".ptxas.txt"), "w") as f:
            f.write("\n".join(l for l in out.splitlines() if "ptxas" in l or "spill" in l) + "\n")
    return obj


def build_lib(force: bool = False) -> str:
    if force or _stale(LIB, _deps(*UNITS)):
        nvcc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
        with ThreadPoolExecutor(len(UNITS)) as pool:  # one nvcc process for each source
            objs = list(pool.map(lambda n: _build_unit(nvcc, n, force), UNITS))
        tmp = _tmp(LIB)
        _run([nvcc, *NVCC_FLAGS[:2], "-shared", *objs, "-o", tmp])
        os.replace(tmp, LIB)
    return LIB


def build_ext(force: bool = False) -> str:
    deps = _deps(*EXT_SOURCES) + [LIB]
    if force or _stale(EXT, deps):
        import torch
        import torch.utils.cpp_extension as ce
        incs = ce.include_paths("cuda") + [sysconfig.get_paths()["include"], INCLUDE]
        libdirs = ce.library_paths("cuda")
        flags = ["-fPIC", "-O2", "-std=c++17", "-DTORCH_EXTENSION_NAME=_tma_dwconv_C",
                 "-DTORCH_API_INCLUDE_EXTENSION_H",
                 f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                 *[f"-I{i}" for i in incs]]

        def unit(name: str) -> str:
            obj = os.path.join(HERE, name.replace(".cpp", ".o"))
            if force or _stale(obj, _deps(name)):
                _run(["g++", "-c", *flags, os.path.join(CSRC, name), "-o", _tmp(obj)])
                os.replace(_tmp(obj), obj)
            return obj

        with ThreadPoolExecutor(len(EXT_SOURCES)) as pool:
            objs = list(pool.map(unit, EXT_SOURCES))
        _run(["g++", "-shared", *objs, "-o", _tmp(EXT), f"-L{HERE}", "-ltdc_sm100",
              "-Wl,-rpath,$ORIGIN", *[f"-L{d}" for d in libdirs],
              "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10_cuda", "-ltorch_cuda",
              "-lcudart"])
        os.replace(_tmp(EXT), EXT)
    return EXT


def build_all(force: bool = False) -> None:
    build_lib(force)
    build_ext(force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
    print(LIB)
    print(EXT)
