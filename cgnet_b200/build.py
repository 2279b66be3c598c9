"""Build libcgnet_b200.so in-tree with nvcc for sm_100a, and _torch_head.so beside it.

    python -m cgnet_b200.build [--force] [--verbose]

The library is plain CUDA C++ behind a C ABI (include/cgnet_b200.h); it does not link against torch.  _torch_head.so is the
torch side of the operators in head.py (autograd nodes in C++); it links against torch and the library, and is bound to the
version of torch it was compiled with.  The library is complete before it is waited for, and a host without torch gets the
library alone.
"""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
SOURCES = ["plan.cu", "unfused.cu", "fused.cu", "fused_tc.cu", "gff_tc.cu", "sh_project.cu", "raycast.cu",
           "layer_norm.cu", "class_scores.cu", "gated_ff.cu"]
LIB = os.path.join(HERE, "libcgnet_b200.so")
BINDING = os.path.join(HERE, "_torch_head.so")
BINDING_SOURCE = "torch_head.cpp"
BINDING_TORCH = os.path.join(HERE, "_torch_head.torch")     # the version of torch the binding was compiled with
HEADER = os.path.join(HERE, "..", "include", "cgnet_b200.h")
# raycast.cu: no fused multiply-add, so that its float64 hit tests round exactly like a host evaluation of the same
# expressions and rays through shared edges pick the same triangle on both sides
EXTRA_FLAGS = {"raycast.cu": ["-fmad=false"]}
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-Xcompiler", "-O2"]


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    raise RuntimeError("nvcc not found")


def _older(product, deps):
    return not os.path.exists(product) or any(os.path.getmtime(d) > os.path.getmtime(product) for d in deps)


def _library_stale():
    return _older(LIB, [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))] + [HEADER])


def _torch_version():
    """The installed torch, None where there is none (the binding is not built then)."""
    try:
        import torch
    except ImportError:
        return None
    return torch.__version__


def _binding_stale(version):
    if version is None:
        return False
    if _older(BINDING, [os.path.join(CSRC, BINDING_SOURCE), HEADER]) or not os.path.exists(BINDING_TORCH):
        return True
    with open(BINDING_TORCH) as f:
        return f.read() != version


def needs_build():
    return _library_stale() or _binding_stale(_torch_version())


def _torch_paths():
    from torch.utils import cpp_extension
    return cpp_extension.include_paths(device_type="cuda"), cpp_extension.library_paths(device_type="cuda")


def _compile_binding(obj_dir):
    """Start the compilation of torch_head.cpp: (object, process).  With the g++ nvcc uses, whatever CXX says: it has to share torch's
    libstdc++."""
    import torch
    obj = os.path.join(obj_dir, BINDING_SOURCE + ".o")
    includes = [f"-I{p}" for p in _torch_paths()[0]] + [f"-I{sysconfig.get_paths()['include']}"]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + includes + \
        ["-c", os.path.join(CSRC, BINDING_SOURCE), "-o", obj]
    return obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _link_binding(obj, version):
    libs = _torch_paths()[1]
    subprocess.check_call(["g++", "-shared", "-o", BINDING, obj, f"-L{HERE}", f"-l:{os.path.basename(LIB)}", "-Wl,-rpath,$ORIGIN"] + [f"-L{p}" for p in libs] +
                          ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"] + [f"-Wl,-rpath,{libs[0]}"])
    with open(BINDING_TORCH, "w") as f:
        f.write(version)


def _finish(src, p, verbose):
    out, _ = p.communicate()
    if p.returncode != 0:
        raise RuntimeError(f"compiling {src} failed:\n{out}")
    if verbose:
        print(out)


def _build_library(obj_dir, verbose):
    flags = list(NVCC_FLAGS)
    if verbose:
        flags += ["-Xptxas", "-v"]
    procs = []
    for src in SOURCES:
        obj = os.path.join(obj_dir, src.replace(".cu", ".o"))
        cmd = [_nvcc()] + flags + EXTRA_FLAGS.get(src, []) + ["-c", os.path.join(CSRC, src), "-o", obj]
        procs.append((src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for src, _, p in procs:
        _finish(src, p, verbose)
    subprocess.check_call([_nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB] + [obj for _, obj, _ in procs])


def build(force=False, verbose=False):
    """Compile every .cu of the package into one shared library (object files in csrc/_obj, compiled in parallel), and the binding
    beside it, each where it is older than its sources."""
    version = _torch_version()
    library, binding = force or _library_stale(), version is not None and (force or _binding_stale(version))
    obj_dir = os.path.join(CSRC, "_obj")
    os.makedirs(obj_dir, exist_ok=True)
    if binding:
        obj, p = _compile_binding(obj_dir)
    if library:
        _build_library(obj_dir, verbose)
    if binding:
        _finish(BINDING_SOURCE, p, verbose)
        _link_binding(obj, version)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
