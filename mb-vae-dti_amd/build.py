"""Build libmbvae_hip.so (gfx950) in-tree with hipcc.  `python mb-vae-dti_amd/build.py [--force]`."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libmbvae_hip.so")
HOST_SRC = os.path.join(CSRC, "host.cpp")                      # host code only: checks, allocation and autograd nodes of a few operators
HOST_OUT = os.path.join(HERE, "mbvae_amd", "_host.so")
SOURCES = ["gemm.hip", "edge_attn.hip", "edge_fused.hip", "rowops.hip", "loss.hip", "diffusion.hip", "eigen.hip", "cycles.hip",
           "gated_norm_f32.hip", "gated_norm_bf16.hip", "gated_norm_f16.hip", "gated_norm.hip", "embedding.hip", "gradclip.hip"]
# No packed-fp32 instructions (v_pk_*_f32) in device code.  Measured on MI355X: the node-path LayerNorm backward
# (ln_res_bwd_kernel<64, 1>), whose compiled form reads its per-row statistics through op_sel'ed packed operands, returned
# rare wrong rows (the low half of one packed subtract behaving as "minus 0" in lanes 48-63) whenever tall-skinny product
# kernels of ANOTHER stream were running on the chip, and never on an idle one; compiled without packed fp32 the same
# source is bit-stable next to them (tools/concurrency_probe.py, tests/test_gpu_concurrency.py).  The train step's time is
# the same with and without (54.5-54.9 ms either way): the row kernels are memory bound and the matrix kernels' epilogues
# do not depend on packed issue.  The host pass does not know the feature and says so; that warning is filtered below.
# A 64-bit count that becomes a 32-bit one without a cast is an error: tensors pass 2^31 values here.
FLAGS = ["-O3", "--offload-arch=gfx950", "-fPIC", "-std=c++17", "-ffp-contract=on", "-Werror=shorten-64-to-32",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def host_command():
    """The compiler call of the Python extension module (g++ against torch's headers; torch's libraries are in the process already
    when it is imported, so their names are all it needs)."""
    import sysconfig
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), "/opt/rocm/include",
           sysconfig.get_paths()["include"]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-w", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            "-DTORCH_EXTENSION_NAME=_host", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-isystem{i}" for i in inc),
            HOST_SRC, "-o", HOST_OUT, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python"]


def build(force=False, verbose=True):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    common = [os.path.join(CSRC, h) for h in ("common.h", "typed.h", "gated_norm.h", "gated_norm_kernels.h")]
    jobs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src.replace(".hip", ".o"))
        if force or _stale(o, [s] + common):
            jobs.append([hipcc, *FLAGS, "-c", s, "-o", o])
    kernels = bool(jobs)
    if force or _stale(HOST_OUT, [HOST_SRC]):
        jobs.insert(0, host_command())

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, stderr=subprocess.PIPE, text=True)
        err = "\n".join(l for l in res.stderr.splitlines() if "'-packed-fp32-ops' is not a recognized feature" not in l)
        if err.strip():
            print(err, file=sys.stderr, flush=True)
        if res.returncode != 0:
            raise subprocess.CalledProcessError(res.returncode, cmd)

    with ThreadPoolExecutor(max_workers=4) as ex:
        list(ex.map(run, jobs))
    objs = [os.path.join(objdir, s.replace(".hip", ".o")) for s in SOURCES]
    if force or kernels or _stale(OUT, objs):
        run([hipcc, "-shared", "-fPIC", "--offload-arch=gfx950", "-o", OUT, *objs])
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(OUT)
