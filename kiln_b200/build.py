"""Builds the CUDA library in-tree for sm_100a: kiln_b200/lib/libkiln_b200.so, and what binds it: the C++ op-set shim and the torch binding.

    python -m kiln_b200.build [--force] [--verbose]

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically and resolves the
one driver entry point it needs (cuTensorMapEncodeTiled) at run time, so it loads on a machine
without a driver; every launch entry point then fails with KB_ERR_DEVICE.
"""
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB_DIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIB_DIR, "libkiln_b200.so")
HOST_LIB = os.path.join(LIB_DIR, "libkiln_engine_ops.so")
BINDING = os.path.join(LIB_DIR, "_kiln_torch.so")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")

NVCC_FLAGS = ["-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
              "-Xcompiler", "-fPIC", "-shared", "-I" + INCLUDE]


def _sources(dirs, exts):
    out = []
    for d in dirs:
        for root, _, files in os.walk(d):
            out += [os.path.join(root, f) for f in files if f.endswith(exts)]
    return out


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False, defines=(), out=None):
    """Compile csrc/abi.cu (which includes every kernel) into the shared library; returns its path."""
    out = out or LIB
    os.makedirs(os.path.dirname(out), exist_ok=True)
    deps = _sources([CSRC, INCLUDE], (".cu", ".cuh", ".h"))
    if force or _stale(out, deps):
        _compile(out, verbose, defines)
    if out == LIB:
        build_binding()                            # ops.py binds some of the library's calls with it
    return out


def _compile(out, verbose, defines):
    cmd = ["nvcc"] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-D" + d for d in defines] + \
          ["-o", out, os.path.join(CSRC, "abi.cu")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose:
        sys.stderr.write(r.stderr)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stderr[-6000:])


def build_host(force=False):
    """Compile the C++ host shim (the engine-facing op set) against the C ABI; returns its path."""
    src = os.path.join(PKG, "host", "gpu_ops.cpp")
    deps = _sources([os.path.join(PKG, "host"), INCLUDE], (".cpp", ".h"))
    if not force and not _stale(HOST_LIB, deps + [LIB]):
        return HOST_LIB
    cmd = ["nvcc", "-O2", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", "-I" + INCLUDE, "-o", HOST_LIB, src,
           "-L" + LIB_DIR, "-lkiln_b200", "-Xlinker", "-rpath", "-Xlinker", "$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("host shim build failed:\n" + r.stderr[-6000:])
    return HOST_LIB


def torch_tag(torch_dir):
    """What the binding is compiled for: it takes the layout of torch's and Python's structures from their headers."""
    with open(os.path.join(torch_dir, "version.py")) as f:
        version = re.search(r"^__version__\s*=\s*['\"]([^'\"]+)", f.read(), flags=re.M).group(1)
    return f"torch {version}, {sysconfig.get_config_var('SOABI')}"


def _built_for(path, tag):
    with open(path, "rb") as f:
        return f"[{tag}]".encode() in f.read()


def build_binding(force=False):
    """Compile the binding of the 4-bit, rotary and dropout calls for torch tensors (a CPython module, no device code); returns its path, or None where
    there is no torch: the library and the C++ shim need none, and without the binding those calls of ops.py refuse."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:
        sys.stderr.write("kiln_b200: no torch here, so its binding is not built\n")
        return None
    src = os.path.join(PKG, "host", "torch_binding.cpp")
    torch_dir = os.path.dirname(spec.origin)
    tag = torch_tag(torch_dir)
    if not force and not _stale(BINDING, [src, os.path.join(INCLUDE, "kiln_b200.h")]) and _built_for(BINDING, tag):
        return BINDING
    os.makedirs(os.path.dirname(BINDING), exist_ok=True)
    inc = os.path.join(torch_dir, "include")
    cuda = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w", f'-DKB_BUILT_FOR="{tag}"', "-I" + inc, "-I" + os.path.join(inc, "torch", "csrc", "api", "include"),
           "-I" + os.path.join(cuda, "include"), "-I" + sysconfig.get_paths()["include"], "-o", BINDING + ".new", src, "-L" + os.path.join(torch_dir, "lib"),
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("torch binding build failed:\n" + r.stderr[-6000:])
    os.replace(BINDING + ".new", BINDING)
    return BINDING


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
    if os.path.exists(os.path.join(PKG, "host", "gpu_ops.cpp")):
        print(build_host(force="--force" in sys.argv))
    if build_binding(force="--force" in sys.argv):
        print(BINDING)
