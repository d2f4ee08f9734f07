"""Build the HIP libraries of the package in-tree with hipcc for gfx950.

Each library is one ``hipcc -shared`` over its sources in ``csrc/``; the output
``.so`` sits next to this file and is what ``_lib.py`` loads.  ``_ops.so`` (host C++, the
operators' torch calls) is built over the library.
"""
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ARCH = os.environ.get("MSD_OFFLOAD_ARCH", "gfx950")

# Packed FP32 VALU ops are disabled for all device code (compiler flag, device pass only).
HIPCC_FLAGS = ["-O3", "-std=c++17", "-fPIC", "-shared", f"--offload-arch={ARCH}",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
               "-Wno-unused-command-line-argument"]

LIBS = {
    "libmsdecode.so": ["csrc/msdecode.hip", "csrc/sample.hip", "csrc/prefill.hip", "csrc/batched.hip",
                       "csrc/xent.hip", "csrc/attn.hip", "csrc/layers.hip", "csrc/paged.hip"],
}


def hipcc():
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found")


def ops_command(out):
    """The host compiler's command for _ops.so, over libmsdecode.so beside it (HIP's headers want to be told their platform
    by a compiler that is not hipcc)."""
    import torch
    base = os.path.dirname(torch.__file__)
    include = [os.path.join(base, "include"), os.path.join(base, "include/torch/csrc/api/include"),
               sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(hipcc())), "include")]
    return [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1",
            "-DTORCH_EXTENSION_NAME=_ops", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[x for i in include for x in ("-isystem", i)], os.path.join(HERE, "csrc/torch_ops.cpp"), "-o", out,
            "-L" + os.path.join(base, "lib"), "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip", "-ltorch_python", "-L" + HERE,
            "-l:libmsdecode.so", "-Wl,-rpath,$ORIGIN"]


def build(verbose=False):
    cc = hipcc()
    for lib, srcs in LIBS.items():
        out = os.path.join(HERE, lib)
        tmp = out + ".tmp"
        cmd = [cc, *HIPCC_FLAGS, "-o", tmp, *[os.path.join(HERE, s) for s in srcs]]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError(f"hipcc failed for {lib}")
        os.replace(tmp, out)
    out = os.path.join(HERE, "_ops.so")
    cmd = ops_command(out + ".tmp")
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("the host compiler failed for _ops.so")
    os.replace(out + ".tmp", out)
    return [os.path.join(HERE, lib) for lib in LIBS] + [out]


if __name__ == "__main__":
    for p in build(verbose=True):
        print("built", p)
