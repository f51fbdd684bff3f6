"""
Build libbgmm_hip.so and libbgmm_ops.so (hipcc, gfx950 only) in-tree next to their sources.

The shared objects are git-ignored but travel to the GPU box with the gpurun
snapshot.  ``build()`` is idempotent: it recompiles only sources newer than
their objects.
"""
import glob
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbgmm_hip.so")
SOURCES = ["api_context.hip", "api_inputs.hip", "api_perm.hip", "api_sweep.hip", "api_group.hip", "api_comm.hip", "kernels_state.hip", "kernels_score.hip", "kernels_prune.hip", "kernels_choice.hip",
           "kernels_resolve.hip", "kernels_rng.hip", "kernels_seq.hip", "kernels_gram.hip", "kernels_home.hip", "kernels_safe.hip",
           "kernels_perm.hip", "kernels_resid.hip"]
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
# every header next to the sources + the public one: editing any of them rebuilds every object
HEADERS = sorted(h for h in glob.glob(os.path.join(CSRC, "*.h")) if not os.path.basename(h).startswith("ops_")) + [os.path.join(INCLUDE, "bgmm.h")]
# the operators on torch tensors (pybgmm_amd.ops): a library of its own, because it has to bind to the HIP runtime that
# torch brings, while libbgmm_hip.so links the system's (a process may hold both)
OPS_LIB = os.path.join(HERE, "libbgmm_ops.so")
OPS_SOURCES = ["ops_common.hip", "ops_groups.hip", "ops_products.hip", "ops_products_f64.hip", "ops_products_f32.hip",
               "ops_products_f16.hip", "ops_products_bf16.hip", "ops_route.hip", "ops_verify.hip"]
OPS_HEADERS = sorted(glob.glob(os.path.join(CSRC, "ops_*.h"))) + [os.path.join(INCLUDE, "bgmm_ops.h")]
# -ffp-contract=off: the sufficient-statistics updates must round product and sum
# separately (bit-identical m / S to the reference); hot loops call fma() explicitly.
# -fvisibility=hidden: the shared object exports the BGMM_API entry points of include/bgmm.h and nothing else.
# -packed-fp32-ops: no packed single-precision arithmetic (some of its forms have given wrong results on this hardware);
# hipcc's host pass does not know the feature and says so, which is harmless.
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fvisibility=hidden",
         "-Wall", "-Wno-unused-result", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def hipcc():
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found: libbgmm_hip.so cannot be built")
    return exe


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False, extra_flags=()):
    """Both libraries; returns the path of libbgmm_hip.so."""
    # -no-hip-rt: libbgmm_ops.so does not link a HIP runtime (include/bgmm_ops.h says which one it binds to)
    _build_one(OPS_LIB, OPS_SOURCES, OPS_HEADERS, ["-no-hip-rt"], force, verbose, extra_flags)
    return _build_one(LIB, SOURCES, HEADERS, [], force, verbose, extra_flags)


def _build_one(lib, sources, headers, link_flags, force, verbose, extra_flags):
    objdir = os.path.join(CSRC, "_obj")
    os.makedirs(objdir, exist_ok=True)
    cc = hipcc()
    jobs = []
    for src in sources:
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src + ".o")
        if force or _stale(o, [s] + headers):
            jobs.append([cc] + FLAGS + list(extra_flags) + ["-c", s, "-o", o])

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed:\n%s\n%s" % (" ".join(cmd), r.stdout))
        return r.stdout

    if jobs:
        with ThreadPoolExecutor(max_workers=4) as ex:
            outs = list(ex.map(run, jobs))
        if verbose:
            for o in outs:
                if o.strip():
                    print(o)
    objs = [os.path.join(objdir, s + ".o") for s in sources]
    if force or jobs or _stale(lib, objs):
        run([cc, "--offload-arch=gfx950", "-shared", "-fPIC"] + link_flags + ["-o", lib] + objs)
    return lib


if __name__ == "__main__":
    import sys
    print(build(force="--force" in sys.argv, verbose=True))
