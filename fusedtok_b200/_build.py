"""In-tree build of the CUDA library (sm_100a only).

``python fusedtok_b200/_build.py`` compiles ``csrc/*.cu`` into
``fusedtok_b200/libfusedtok_b200.so`` with nvcc. The library is the whole
product: there is no other backend and no CPU fallback, so importing the
package without it fails.
"""

import os
import re
import subprocess
import sys
import sysconfig
import time

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libfusedtok_b200.so")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))
OBJECTS = os.path.join(HERE, "build")       # one object per source and variant, kept between builds

NVCC_FLAGS = [
    "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
    "-Xcompiler", "-fPIC",
]
LINK_FLAGS = ["-shared", "-cudart", "static", "-gencode", "arch=compute_100a,code=sm_100a"]


# The self-checking variant (tests/test_bounds_build_gpu.py): same sources with -DFTK_BOUNDS.
BOUNDS_LIB = os.path.join(HERE, "libfusedtok_b200_bounds.so")


def _includes(path, seen=None):
    """`path` and every file it includes with quotes, directly or not."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path in seen or not os.path.exists(path):
        return seen
    seen.add(path)
    with open(path) as f:
        for name in re.findall(r'^\s*#include "([^"]+)"', f.read(), flags=re.M):
            _includes(os.path.join(os.path.dirname(path), name), seen)
    return seen


def _out_of_date(target, source):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in _includes(source))


def stale(target=None):
    target = target or LIB
    return any(_out_of_date(target, os.path.join(CSRC, s)) for s in SOURCES)


def _compile(variants, force=False, verbose=False):
    """Bring the objects of `variants` [(defines, target)] up to date, every source in an nvcc of its own side by
    side, and link each variant's library. What is built is dated from when the build began: an edit made meanwhile
    leaves it out of date."""
    os.makedirs(OBJECTS, exist_ok=True)
    began = time.time()
    jobs, linked = [], []
    for defines, target in variants:
        tag = "".join("_" + re.sub(r"\W", "_", d) for d in sorted(defines))
        objects = []
        for s in SOURCES:
            source, obj = os.path.join(CSRC, s), os.path.join(OBJECTS, s[:-3] + tag + ".o")
            objects.append(obj)
            if force or _out_of_date(obj, source):
                jobs.append((os.path.getsize(source), ["nvcc"] + NVCC_FLAGS + ["-D" + d for d in defines]
                             + (["-Xptxas", "-v"] if verbose else []) + ["-c", source, "-o", obj]))
        linked.append((objects, target))
    jobs.sort(key=lambda j: -j[0])                    # the longest first
    running, failed = [], []
    while jobs or running:
        while jobs and len(running) < max(2, os.cpu_count() or 2):
            cmd = jobs.pop(0)[1]
            running.append((cmd, subprocess.Popen(cmd)))
        cmd, job = running.pop(0)
        try:
            if job.wait(timeout=1) != 0:
                failed.append(cmd[-1])
            else:
                os.utime(cmd[-1], (began, began))
        except subprocess.TimeoutExpired:
            running.append((cmd, job))
    if failed:
        raise RuntimeError("nvcc failed for " + ", ".join(failed))
    for objects, target in linked:
        subprocess.check_call(["nvcc"] + LINK_FLAGS + objects + ["-o", target])
        os.utime(target, (began, began))


# The module that makes plain calls straight from torch tensors (csrc/tensor_calls.cpp). An accelerator of the Python
# wrappers, not another way to compute: without it every call takes the wrappers' way.
BINDING = os.path.join(HERE, "_tensors.so")


def build_binding(force=False):
    """Compile the module with the C++ headers of the installed torch; nothing to do without torch."""
    source = os.path.join(CSRC, "tensor_calls.cpp")
    stamp = os.path.join(OBJECTS, "tensor_calls.torch")      # the torch it was built for
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError:
        return None
    built_for = open(stamp).read() if os.path.exists(stamp) else ""
    if not force and built_for == torch.__version__ and not _out_of_date(BINDING, source):
        return BINDING
    began = time.time()
    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME") or cpp_extension.CUDA_HOME or "/usr/local/cuda"
    cmd = ["g++", "-O2", "-std=c++20", "-fPIC", "-shared", source, "-o", BINDING]
    for d in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
              os.path.join(cuda, "include"), sysconfig.get_paths()["include"]):
        cmd += ["-I", d]
    cmd += ["-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if subprocess.call(cmd) != 0:
        if os.path.exists(BINDING):
            os.remove(BINDING)
        print("fusedtok_b200: %s was not built; calls take the Python wrappers' way" % BINDING)
        return None
    os.utime(BINDING, (began, began))
    os.makedirs(OBJECTS, exist_ok=True)
    with open(stamp, "w") as f:
        f.write(torch.__version__)
    return BINDING


def build_all(force=False):
    """The product and the self-checking variant, whichever is out of date, compiled side by side."""
    _compile([(d, t) for d, t in (((), LIB), (("FTK_BOUNDS",), BOUNDS_LIB)) if force or stale(t)], force)
    build_binding(force)
    return LIB


def build(force=False, verbose=False, defines=(), out=None):
    """Compile the library. `defines` / `out` produce a variant build next to the product (for example
    ``defines=["FTK_TIMELINE"]``: per-CTA timestamps in the tensor-core decode kernel, read back with
    ``ftk_debug_timeline``); the product itself is always built without defines."""
    target = out or LIB
    if not defines:
        build_binding(force)
    if not force and not defines and not stale():
        return LIB
    _compile([(tuple(defines), target)], force, verbose)
    return target


if __name__ == "__main__":
    # python fusedtok_b200/_build.py [--force] [-v] [-DNAME ...] [--out path] | --all
    if "--all" in sys.argv:
        print(build_all(force="--force" in sys.argv))
        sys.exit(0)
    defs = [a[2:] for a in sys.argv[1:] if a.startswith("-D")]
    out_path = sys.argv[sys.argv.index("--out") + 1] if "--out" in sys.argv else None
    if defs and not out_path:
        raise SystemExit("a build with -D defines needs --out: the product library is built without defines")
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, defines=defs, out=out_path))
