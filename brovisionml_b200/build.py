"""Build libbvml_dsine.so (the CUDA kernels + C ABI) for sm_100a, in-tree.

    python brovisionml_b200/build.py [--ptxas]

(Run it by path: importing the package loads the library, which may be stale
or missing before this script has run.)

Compiles each brovisionml_b200/csrc/*.cu with nvcc for
``-gencode arch=compute_100a,code=sm_100a`` (B200 only) and links them into
``brovisionml_b200/_lib/libbvml_dsine.so``, and csrc/blocks/*.cu (the
feed-forward operators, include/bvml_blocks.h) into ``_lib/libbvml_blocks.so``,
with their Python binding (csrc/blocks/blocks_torch.cpp) for this torch and Python in
``_lib/_blocks_torch.<Python's ABI>.torch<version>.so``.
The C++ drop-in bridge
(csrc/dsine_ops_b200.cpp) is compiled into ``_lib/libbvml_dsine_bridge.so``
against the stand-in brotensor header, to prove that it builds.
Rebuilds only what changed (source / header mtimes).
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "_lib")
OBJ_DIR = os.path.join(HERE, "_build")
LIB = os.path.join(LIB_DIR, "libbvml_dsine.so")
# The same sources with -DBVML_CHECKED: every kernel tests its indices and TMA
# coordinates before each access and records failures (bvml_check_word); the
# GPU tests run the odd shapes through it.
CHECKED_LIB = os.path.join(LIB_DIR, "libbvml_dsine_checked.so")
BLOCKS = os.path.join(CSRC, "blocks")
BLOCKS_LIB = os.path.join(LIB_DIR, "libbvml_blocks.so")
BLOCKS_CHECKED_LIB = os.path.join(LIB_DIR, "libbvml_blocks_checked.so")
BRIDGE = os.path.join(LIB_DIR, "libbvml_dsine_bridge.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
              "--expt-relaxed-constexpr", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is needed to build brovisionml_b200")


def torch_version() -> str | None:
    """torch.__version__ without importing torch; None where there is no torch."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:
        return None
    with open(os.path.join(os.path.dirname(spec.origin), "version.py")) as f:
        m = re.search(r"^__version__\s*=\s*['\"]([^'\"]+)['\"]", f.read(), re.M)
    return m.group(1) if m else None


def blocks_torch_path(torch_ver: str) -> str:
    """The feed-forward operators' Python binding for this Python and a torch, whose C++
    interfaces differ from version to version: one file each, so that none is loaded by
    another, and a new torch or Python has its own built."""
    abi = sysconfig.get_config_var("SOABI")
    return os.path.join(LIB_DIR, f"_blocks_torch.{abi}.torch{torch_ver}.so")


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, ptxas_info: bool = False) -> str:
    """Compile (if stale) and return the path of libbvml_dsine.so. The refinement's
    libraries come first and need nvcc and a C++ compiler alone; the feed-forward
    operators' library next (CUDA 12.9: 32-byte stores), their binding last, and only where
    torch is installed."""
    nvcc = _nvcc()
    os.makedirs(LIB_DIR, exist_ok=True)
    os.makedirs(OBJ_DIR, exist_ok=True)
    headers = (glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h"))
               + glob.glob(os.path.join(ROOT, "include", "*.h")))

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(os.path.basename(cmd[0]) + " failed:\n" + " ".join(cmd) + "\n" +
                               r.stdout + r.stderr)
        return r.stdout + r.stderr

    def libraries(sources, deps, prefix, lib, checked_lib):
        """The sources' objects and checked objects (all at once), and a library of each."""
        jobs, objs, cobjs = [], [], []
        for src in sources:
            name = prefix + os.path.basename(src)[:-3] + ".o"
            obj, cobj = os.path.join(OBJ_DIR, name), os.path.join(OBJ_DIR, "checked_" + name)
            objs.append(obj)
            cobjs.append(cobj)
            if _stale(obj, [src] + deps) or ptxas_info:
                jobs.append([nvcc] + ARCH + NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_info else [])
                            + ["-c", src, "-o", obj])
            if _stale(cobj, [src] + deps):
                jobs.append([nvcc] + ARCH + NVCC_FLAGS + ["-DBVML_CHECKED", "-c", src, "-o", cobj])
        with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
            for out in ex.map(run, jobs):
                if verbose or ptxas_info:
                    sys.stdout.write(out)
        for target, parts in ((lib, objs), (checked_lib, cobjs)):
            if _stale(target, parts + [__file__]):
                # Shared cudart: callers (torch, or a brotensor runtime) hand in stream
                # handles created by THEIR CUDA runtime; one shared runtime instance
                # per process is what makes those handles valid here too.
                run([nvcc] + ARCH + ["-shared", "-cudart", "shared", "-o", target] + parts +
                    ["-Xlinker", "-rpath,/usr/local/cuda/lib64"])

    libraries(sorted(glob.glob(os.path.join(CSRC, "*.cu"))), headers, "", LIB, CHECKED_LIB)
    _build_bridge(nvcc, headers, run)
    # the feed-forward operators: a library of their own, so that the ABI of
    # libbvml_dsine.so stays as it is
    libraries(sorted(glob.glob(os.path.join(BLOCKS, "*.cu"))),
              headers + glob.glob(os.path.join(BLOCKS, "*.cuh")) +
              glob.glob(os.path.join(BLOCKS, "*.h")), "blocks_", BLOCKS_LIB, BLOCKS_CHECKED_LIB)
    _build_binding(nvcc, headers, run)
    return LIB


def _build_bridge(nvcc, headers, run):
    bridge_src = os.path.join(CSRC, "dsine_ops_b200.cpp")
    if not os.path.exists(bridge_src):
        return
    deps = [bridge_src, LIB] + headers + glob.glob(os.path.join(CSRC, "brotensor_shim", "*", "*.h"))
    if _stale(BRIDGE, deps):
        cxx = os.environ.get("CXX") or shutil.which("g++") or "g++"
        cuda = os.path.dirname(os.path.dirname(nvcc))
        run([cxx, "-O2", "-std=c++20", "-fPIC", "-shared", "-Wall", "-Wextra",
             "-I" + os.path.join(CSRC, "brotensor_shim"), "-I" + os.path.join(ROOT, "include"),
             "-I" + os.path.join(cuda, "include"), "-DBVML_SHIM_CUDA", bridge_src, "-o", BRIDGE,
             "-L" + LIB_DIR, "-lbvml_dsine", "-Wl,-rpath,$ORIGIN",
             "-L" + os.path.join(cuda, "lib64"), "-lcudart", "-Wl,--exclude-libs,ALL"])


def _build_binding(nvcc, headers, run):
    version = torch_version()
    if version is None:
        print("no torch here: the feed-forward operators' Python binding is left out",
              file=sys.stderr)
        return
    src, target = os.path.join(BLOCKS, "blocks_torch.cpp"), blocks_torch_path(version)
    if _stale(target, [src, BLOCKS_LIB, __file__] + headers):
        torch_dir = os.path.dirname(importlib.util.find_spec("torch").origin)
        cuda = os.path.dirname(os.path.dirname(nvcc))
        run([os.environ.get("CXX") or shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC",
             "-shared", "-fvisibility=hidden", "-DUSE_CUDA",
             "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(cuda, "include"),
             "-isystem", os.path.join(torch_dir, "include"),
             "-isystem", os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
             "-I" + sysconfig.get_path("include"), src, "-o", target,
             "-L" + LIB_DIR, "-lbvml_blocks", "-Wl,-rpath,$ORIGIN",
             "-L" + os.path.join(torch_dir, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu",
             "-ltorch_cuda", "-lc10", "-lc10_cuda",
             "-Wl,-rpath," + os.path.join(torch_dir, "lib")])


if __name__ == "__main__":
    print(build(verbose=True, ptxas_info="--ptxas" in sys.argv))
