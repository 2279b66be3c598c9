"""Build libcgnet_b200.so in-tree with nvcc for sm_100a, and _torch_head.so beside it.

    python -m cgnet_b200.build [--force] [--verbose]

The library is plain CUDA C++ behind a C ABI (include/cgnet_b200.h); it does not link against torch.  _torch_head.so is the
torch side of the operators in head.py (autograd nodes in C++); it links against torch and the library.
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


def needs_build():
    if not os.path.exists(LIB) or not os.path.exists(BINDING):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(BINDING))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "cgnet_b200.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def _torch_paths():
    from torch.utils import cpp_extension
    return cpp_extension.include_paths(device_type="cuda"), cpp_extension.library_paths(device_type="cuda")


def _compile_binding(obj_dir):
    """Start the compilation of torch_head.cpp: (source, object, process).  With the g++ nvcc uses, whatever CXX says: it has to
    share torch's libstdc++."""
    import torch
    src, obj = "torch_head.cpp", os.path.join(obj_dir, "torch_head.cpp.o")
    includes = [f"-I{p}" for p in _torch_paths()[0]] + [f"-I{sysconfig.get_paths()['include']}"]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + includes + \
        ["-c", os.path.join(CSRC, src), "-o", obj]
    return src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _link_binding(obj):
    libs = _torch_paths()[1]
    subprocess.check_call(["g++", "-shared", "-o", BINDING, obj, f"-L{HERE}", f"-l:{os.path.basename(LIB)}", "-Wl,-rpath,$ORIGIN"] + [f"-L{p}" for p in libs] +
                          ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"] + [f"-Wl,-rpath,{libs[0]}"])


def build(force=False, verbose=False):
    """Compile every .cu of the package into one shared library (object files in csrc/_obj, compiled in parallel)."""
    if not force and not needs_build():
        return LIB
    obj_dir = os.path.join(CSRC, "_obj")
    os.makedirs(obj_dir, exist_ok=True)
    flags = list(NVCC_FLAGS)
    if verbose:
        flags += ["-Xptxas", "-v"]
    procs = [_compile_binding(obj_dir)]
    for src in SOURCES:
        obj = os.path.join(obj_dir, src.replace(".cu", ".o"))
        cmd = [_nvcc()] + flags + EXTRA_FLAGS.get(src, []) + ["-c", os.path.join(CSRC, src), "-o", obj]
        procs.append((src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    objs = []
    binding_obj = procs[0][1]
    for src, obj, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"compiling {src} failed:\n{out}")
        if verbose:
            print(out)
        if obj != binding_obj:
            objs.append(obj)
    cmd = [_nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB] + objs
    subprocess.check_call(cmd)
    _link_binding(binding_obj)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
