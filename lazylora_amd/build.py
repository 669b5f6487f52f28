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
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as exc:  # no such compiler
        return 127, str(exc)
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
    translation units in parallel, objects under _build/). Returns the library path. LIB needs hipcc
    alone and is linked whatever becomes of the module, which needs torch's and Python's headers and a
    host compiler; RuntimeError, afterwards, if the module could not be built."""
    from concurrent.futures import ThreadPoolExecutor
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    compile_flags = [f for f in FLAGS if f != "-shared"]
    jobs = []
    for src in SOURCES:
        obj = os.path.join(objdir, os.path.splitext(src)[0] + ".o")
        jobs.append(([HIPCC] + compile_flags + FILE_FLAGS.get(src, []) + ["-c", os.path.join(CSRC, src), "-o", obj],
                     obj))
    module, trouble = None, ""
    try:
        module = _autograd_commands(objdir)
    except ImportError as exc:
        trouble = str(exc)
    commands = [cmd for cmd, _ in jobs] + ([module[0]] if module else [])
    if verbose:
        for cmd in commands:
            print(" ".join(cmd), flush=True)
    with ThreadPoolExecutor(max_workers=min(len(commands), os.cpu_count() or 1, 16)) as ex:
        results = list(ex.map(_run, commands))
    for (cmd, _), (rc, err) in zip(jobs, results):
        if rc != 0:
            raise RuntimeError(f"hipcc failed ({rc}) on {cmd[-3]}:\n{err}")
        if verbose and err:
            print(err, file=sys.stderr)
    _link([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC"] + [o for _, o in jobs]
          + ["-Wl,-soname," + os.path.basename(LIB)], LIB)
    if module:
        (cmd, obj, out, libs), (rc, trouble) = module, results[-1]
        if rc == 0:
            _link([cmd[0], "-shared", "-fPIC", obj] + libs, out)
            return LIB
    raise RuntimeError(f"{os.path.basename(LIB)} is built, but not the autograd module over it ({AUTOGRAD}, the "
                       f"dense operators' Python entry points):\n{trouble}")


def _link(cmd, out):
    """Link into a file beside `out` and move it there, so that a running process keeps what it has loaded."""
    tmp = out + ".tmp"
    rc, err = _run(cmd + ["-o", tmp])
    if rc != 0:
        raise RuntimeError(f"link of {os.path.basename(out)} failed ({rc}):\n{err}")
    os.replace(tmp, out)


if __name__ == "__main__":
    print(build(verbose=True))
