"""Build the gfx950 HIP library in-tree: lazylora_amd/liblazylora_mxfp4.so.

hipcc cross-compiles for gfx950 without a GPU, so this runs on any host with ROCm. The
library is one shared object with a plain C ABI (include/lazylora_mxfp4.h); Python loads it
with ctypes and passes torch device pointers.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liblazylora_mxfp4.so")
AUTOGRAD = "_dense_autograd"  # the dense operators' autograd functions: a Python module over LIB
SOURCES = ["capi.hip", "mx_forward.hip", "mx_backward.hip", "mx_misc.hip", "mx_router.hip", "mx_lora.hip",
           "mx_dense.hip", "mx_rows.hip"]

# per-file flags: the transposed products keep their accumulators in VGPRs (the MFMA's VGPR
# form); with the default heuristics the compiler splits them over AGPRs and VGPRs and shuffles
# them with v_accvgpr moves inside the main loop
FILE_FLAGS = {"mx_backward.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"]}

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    # never emit packed-fp32 VALU ops (v_pk_add/mul/fma_f32)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
    f"-I{os.path.join(ROOT, 'include')}",
]


def _run(cmd):
    res = subprocess.run(cmd, capture_output=True, text=True)
    err = "\n".join(l for l in res.stderr.splitlines() if "packed-fp32-ops" not in l and l.strip())
    return res.returncode, err


def _autograd_commands(objdir):
    """(compile command, object, module path, link options) of the autograd module: host C++ against the
    installed torch, linked to LIB beside it."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    root = os.path.dirname(torch.__file__)
    obj = os.path.join(objdir, AUTOGRAD + ".o")
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                os.path.join(os.path.dirname(os.path.dirname(HIPCC)), "include"), sysconfig.get_paths()["include"]]
    cmd = ([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1",
            "-DUSE_ROCM=1", f"-DTORCH_EXTENSION_NAME={AUTOGRAD}",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
           + [f"-isystem{d}" for d in includes]
           + ["-c", os.path.join(CSRC, "dense_autograd.cpp"), "-o", obj])
    out = os.path.join(HERE, AUTOGRAD + sysconfig.get_config_var("EXT_SUFFIX"))
    libs = [f"-L{d}" for d in cpp_extension.library_paths()] + [
        "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lc10_hip", LIB, "-Wl,-rpath,$ORIGIN"]
    return cmd, obj, out, libs


def build(verbose: bool = False) -> str:
    """Compile every source into LIB, and the autograd module over it (always recompiles; the
    translation units in parallel, objects under _build/). Returns the library path."""
    from concurrent.futures import ThreadPoolExecutor
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    compile_flags = [f for f in FLAGS if f != "-shared"]
    jobs = []
    for src in SOURCES:
        obj = os.path.join(objdir, os.path.splitext(src)[0] + ".o")
        jobs.append(([HIPCC] + compile_flags + FILE_FLAGS.get(src, []) + ["-c", os.path.join(CSRC, src), "-o", obj],
                     obj))
    auto_cmd, auto_obj, auto_out, auto_libs = _autograd_commands(objdir)
    jobs.append((auto_cmd, auto_obj))
    if verbose:
        for cmd, _ in jobs:
            print(" ".join(cmd), flush=True)
    with ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 1, 16)) as ex:
        results = list(ex.map(lambda j: _run(j[0]), jobs))
    for (cmd, _), (rc, err) in zip(jobs, results):
        if rc != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({rc}) on {cmd[-3]}:\n{err}")
        if verbose and err:
            print(err, file=sys.stderr)
    tmp = LIB + ".tmp"
    rc, err = _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC"] + [o for _, o in jobs if o != auto_obj]
                   + ["-Wl,-soname," + os.path.basename(LIB), "-o", tmp])
    if rc != 0:
        raise RuntimeError(f"link failed ({rc}):\n{err}")
    os.replace(tmp, LIB)
    tmp = auto_out + ".tmp"
    rc, err = _run([auto_cmd[0], "-shared", "-fPIC", auto_obj] + auto_libs + ["-o", tmp])
    if rc != 0:
        raise RuntimeError(f"link failed ({rc}):\n{err}")
    os.replace(tmp, auto_out)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
