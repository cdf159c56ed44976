"""Build the sqrt-block attention shared library in-tree with nvcc (sm_100a).

    python -m llm_training_b200.build [--force] [--debug]

Produces ``llm_training_b200/lib/libsqrtblock.so`` from ``csrc/*.cu``.  The
library exports the C ABI of ``include/sqrtblock.h`` and links the CUDA
runtime statically, so it depends only on the driver at run time.  And
``lib/sqb_torch.so`` from ``csrc/torch_binding.cpp`` (g++, PyTorch's headers): the
eager PyTorch binding of the post-training operators, left out (with a warning) where
PyTorch or the compiler is not there.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
BUILD = os.path.join(PKG, "_build")
LIBDIR = os.path.join(PKG, "lib")
LIBNAME = "libsqrtblock.so"
LIBPATH = os.path.join(LIBDIR, LIBNAME)
BINDING = "sqb_torch"
BINDINGPATH = os.path.join(LIBDIR, BINDING + ".so")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the sqrt-block CUDA library cannot be built")


def _flags(debug: bool):
    f = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC,-O3", "-I", INCLUDE, "-I", CSRC,
         "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"] + ARCH_FLAGS
    if debug:
        f += ["-DSQB_DEBUG=1"]
    return f


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _torch():
    """(folder, version) of the installed PyTorch, which is not imported; None without one."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    folder = spec.submodule_search_locations[0]
    try:
        return folder, importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return folder, "of unknown version"


def _binding_command(torch_dir: str, out: str):
    """g++ command of the PyTorch binding."""
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path()))), "include")
    headers = [os.path.join(torch_dir, "include"),
               os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"), cuda,
               sysconfig.get_paths()["include"]]
    return ([os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared",
             "-fvisibility=hidden", f"-DTORCH_EXTENSION_NAME={BINDING}", "-I", INCLUDE]
            + [f for h in headers for f in ("-isystem", h)]
            + [os.path.join(CSRC, "torch_binding.cpp"), "-o", out,
               "-L", os.path.join(torch_dir, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
               "-ltorch", "-ltorch_python"])


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, debug: bool = False, verbose: bool = False) -> str:
    """Compile every .cu for sm_100a, link the shared library and, where PyTorch is, build its
    binding; returns the library's path."""
    nvcc = nvcc_path()
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    srcs = _sources()
    hdrs = _headers()
    flags = _flags(debug)
    objs = []
    jobs = []
    for s in srcs:
        obj = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [s] + hdrs + [__file__]):
            jobs.append([nvcc, *flags, "-c", s, "-o", obj])

    # the binding belongs to a PyTorch and a Python
    torch = _torch()
    made_for = f"{torch} {sysconfig.get_config_var('SOABI')}"
    stamp = os.path.join(BUILD, BINDING + ".stamp")
    binding_src = os.path.join(CSRC, "torch_binding.cpp")
    binding_tmp = BINDINGPATH + ".tmp"
    new_binding = (force or torch is None or _stale(BINDINGPATH, [binding_src] + hdrs + [__file__])
                   or not os.path.exists(stamp) or open(stamp).read() != made_for)

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({' '.join(cmd)}):\n{r.stdout}\n{r.stderr}")
        return r.stdout + r.stderr

    with cf.ThreadPoolExecutor(max_workers=max(1, min(len(jobs) + 1, os.cpu_count() or 1))) as ex:
        binding = None
        if new_binding:
            # whatever comes of it, an older one does not stay beside a newer library
            for old in (BINDINGPATH, stamp):
                if os.path.exists(old):
                    os.remove(old)
            if torch is not None:
                binding = ex.submit(run, _binding_command(torch[0], binding_tmp))
        for out in ex.map(run, jobs):
            if verbose and out.strip():
                print(out, flush=True)
    if force or _stale(LIBPATH, objs):
        tmp = LIBPATH + ".tmp"
        run([nvcc, *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", tmp, *objs])
        os.replace(tmp, LIBPATH)
    # the library is there; now the binding's outcome
    why = "PyTorch not found" if torch is None else None
    if binding is not None:
        try:
            out = binding.result()
        except FileNotFoundError as e:
            why = f"no C++ compiler ({e})"
        else:
            if verbose and out.strip():
                print(out, flush=True)
            os.replace(binding_tmp, BINDINGPATH)
            with open(stamp, "w") as f:
                f.write(made_for)
    if why:
        warnings.warn(f"{why}: {BINDINGPATH} is not built, which eager calls of the post-training "
                      "operators need", RuntimeWarning, stacklevel=2)
    return LIBPATH


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--debug", action="store_true", help="build with device-side checks")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args(argv)
    print(build(force=a.force, debug=a.debug, verbose=a.verbose))


if __name__ == "__main__":
    sys.exit(main())
