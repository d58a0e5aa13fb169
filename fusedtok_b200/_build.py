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


def _recipe(cmd):
    """What decides on the result of `cmd` beside the sources: the command, wherever this tree lies, and its compiler's
    version. None without the compiler: what is there then counts as made by it."""
    try:
        version = subprocess.run([cmd[0], "--version"], stdout=subprocess.PIPE, text=True, check=True).stdout
    except FileNotFoundError:
        return None
    return "\n".join(a.replace(HERE, ".") for a in cmd) + "\n" + version


def _stamp(target):
    """File that holds the recipe `target` was made by."""
    return os.path.join(OBJECTS, os.path.basename(target) + ".recipe")


def _made_by(target, recipe):
    if recipe is None or not os.path.exists(target) or not os.path.exists(_stamp(target)):
        return recipe is None and os.path.exists(target)
    with open(_stamp(target)) as f:
        return f.read() == recipe


def _run(jobs, began):
    """Run `jobs` [(target, command, recipe)] side by side. What is built is dated from when the build began: an edit
    made meanwhile leaves it out of date."""
    jobs, running, failed = list(jobs), [], []
    while jobs or running:
        while jobs and len(running) < max(2, os.cpu_count() or 2):
            target, cmd, recipe = jobs.pop(0)
            if os.path.exists(_stamp(target)):
                os.remove(_stamp(target))                 # (until the command has succeeded)
            running.append((target, recipe, subprocess.Popen(cmd)))
        target, recipe, job = running.pop(0)
        try:
            if job.wait(timeout=1) != 0:
                failed.append(target)
                continue
            os.utime(target, (began, began))
            with open(_stamp(target), "w") as f:
                f.write(recipe)
        except subprocess.TimeoutExpired:
            running.append((target, recipe, job))
    if failed:
        raise RuntimeError("building failed for " + ", ".join(failed))


def _compile(variants, force=False, verbose=False):
    """Bring the libraries of `variants` [(defines, target)] up to date: objects whose source, included files, command or
    compiler changed, every source in an nvcc of its own side by side, then the libraries whose objects or command did.
    `verbose` compiles all objects, to report on each."""
    os.makedirs(OBJECTS, exist_ok=True)
    began = time.time()
    jobs, links = [], []
    for defines, target in variants:
        tag = "".join("_" + re.sub(r"\W", "_", d) for d in sorted(defines))
        objects = []
        for s in SOURCES:
            source, obj = os.path.join(CSRC, s), os.path.join(OBJECTS, s[:-3] + tag + ".o")
            objects.append(obj)
            cmd = ["nvcc"] + NVCC_FLAGS + ["-D" + d for d in defines] + ["-c", source, "-o", obj]
            recipe = _recipe(cmd)
            if force or verbose or not _made_by(obj, recipe) or _out_of_date(obj, source):
                jobs.append((os.path.getsize(source), (obj, cmd + (["-Xptxas", "-v"] if verbose else []), recipe)))
        links.append((objects, target))
    jobs.sort(key=lambda j: -j[0])                    # the longest first
    _run([j for _, j in jobs], began)
    built = {j[0] for _, j in jobs}
    for objects, target in links:
        cmd = ["nvcc"] + LINK_FLAGS + objects + ["-o", target]
        recipe = _recipe(cmd)
        if built.intersection(objects) or not _made_by(target, recipe) or any(os.path.getmtime(o) > os.path.getmtime(target) for o in objects):
            _run([(target, cmd, recipe)], began)


# The module that makes plain calls straight from torch tensors (csrc/tensor_calls.cpp). An accelerator of the Python
# wrappers, not another way to compute: without it every call takes the wrappers' way.
BINDING = os.path.join(HERE, "_tensors.so")


def build_binding(force=False):
    """Compile the module with the C++ headers of the installed torch; nothing to do without torch."""
    source = os.path.join(CSRC, "tensor_calls.cpp")
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError:
        return None
    began = time.time()
    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME") or cpp_extension.CUDA_HOME or "/usr/local/cuda"
    cmd = ["g++", "-O2", "-std=c++20", "-fPIC", "-shared", source, "-o", BINDING]
    for d in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
              os.path.join(cuda, "include"), sysconfig.get_paths()["include"]):
        cmd += ["-I", d]
    cmd += ["-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    recipe = _recipe(cmd + [torch.__version__])
    if not force and _made_by(BINDING, recipe) and not _out_of_date(BINDING, source):
        return BINDING
    os.makedirs(OBJECTS, exist_ok=True)
    try:
        _run([(BINDING, cmd, recipe)], began)
    except RuntimeError:
        if os.path.exists(BINDING):
            os.remove(BINDING)
        print("fusedtok_b200: %s was not built; calls take the Python wrappers' way" % BINDING)
        return None
    return BINDING


def build_all(force=False):
    """The product and the self-checking variant, whichever is out of date, compiled side by side."""
    _compile([((), LIB), (("FTK_BOUNDS",), BOUNDS_LIB)], force)
    build_binding(force)
    return LIB


def build(force=False, verbose=False, defines=(), out=None):
    """Compile the library. `defines` / `out` produce a variant build next to the product (for example
    ``defines=["FTK_TIMELINE"]``: per-CTA timestamps in the tensor-core decode kernel, read back with
    ``ftk_debug_timeline``); the product itself is always built without defines."""
    target = out or LIB
    if not defines:
        build_binding(force)
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
