"""Compile the CUDA library (libktir_b200.so) in-tree for sm_100a, and the
serving operators' Python binding (_serving.so), which calls it, where torch is
installed.

    python -m ktir_cpu_b200.build          # or build() from Python

nvcc cross-compiles without a GPU, so this runs on CPU-only hosts too.
"""

from __future__ import annotations

import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libktir_b200.so")
BINDING_SRC = os.path.join(CSRC, "serving_binding.cpp")
BINDING = os.path.join(HERE, "_serving.so")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _newer(target, deps) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(p) <= t for p in deps)


def _torch():
    """The installed torch's folder, or None; it is not imported."""
    spec = importlib.util.find_spec("torch")
    return spec.submodule_search_locations[0] if spec else None


def _made_for() -> str:
    """What a binding fits: it is compiled against torch's and Python's own headers."""
    return f"torch {importlib.metadata.version('torch')}, python {sys.version_info[0]}.{sys.version_info[1]}"


def _stamp() -> str:
    return os.path.join(HERE, "_build", "serving.txt")


def _binding_up_to_date(headers) -> bool:
    if not _newer(BINDING, [BINDING_SRC] + headers) or not os.path.exists(_stamp()):
        return False
    with open(_stamp()) as f:
        return f.read() == _made_for()


def up_to_date() -> bool:
    headers = glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    return _newer(LIB, sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + headers) and \
        (_torch() is None or _binding_up_to_date(headers))


def _compile_binding():
    """The binding's object file and the process that compiles it."""
    import sysconfig
    inc = os.path.join(_torch(), "include")
    obj = os.path.join(HERE, "_build", "serving_binding.o")
    includes = [inc, os.path.join(inc, "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
                os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-c", BINDING_SRC, "-o", obj]
    for p in includes:
        cmd += ["-isystem", p]
    return obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)


def _link_binding(obj):
    cmd = ["g++", "-shared", "-o", BINDING + ".tmp", obj, "-L", HERE, "-l:" + os.path.basename(LIB),
           "-Wl,-rpath,$ORIGIN"]
    cmd += ["-L", os.path.join(_torch(), "lib")]
    # torch's libraries are in the process by the time the binding is imported
    cmd += ["-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda"]
    subprocess.check_call(cmd)
    os.replace(BINDING + ".tmp", BINDING)
    with open(_stamp(), "w") as f:
        f.write(_made_for())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    objs = []
    nvcc = _nvcc()
    tmp = os.path.join(HERE, "_build")
    os.makedirs(tmp, exist_ok=True)
    procs = []
    for src in sources():
        obj = os.path.join(tmp, os.path.basename(src) + ".o")
        cmd = [nvcc, *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
               "-I", os.path.join(HERE, "..", "include"), "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    binding_obj = None
    if _torch():                          # the library alone needs none
        binding_obj, binding = _compile_binding()
        procs.append((BINDING_SRC, binding))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0 or verbose:
            sys.stderr.write(out.decode())
        if p.returncode != 0:
            failed.append(src)
    if failed:
        raise RuntimeError(f"nvcc failed for {failed}")
    tmp_lib = LIB + ".tmp"
    subprocess.check_call([nvcc, *ARCH, "-shared", "-o", tmp_lib, *objs, "-lcudart"])
    os.replace(tmp_lib, LIB)
    if binding_obj:
        _link_binding(binding_obj)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
