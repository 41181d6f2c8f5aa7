"""Build libfa_sm100.so (the sm_100a kernels + C ABI) in-tree with nvcc.

    python fused-attention_b200/build.py            # incremental build
    python fused-attention_b200/build.py --force    # rebuild everything
    python fused-attention_b200/build.py --verbose  # also print ptxas register/smem usage

build_ops() compiles csrc/fa_torch.cpp, the native torch binding of the operators around attention, into
attention/_fa_torch.so against the installed torch; it links libfa_sm100.so next to it.

The shared library lands next to the Python package (attention/libfa_sm100.so), so it travels
with the source tree.  Objects go to _build/ (not committed).

build_stall_test() compiles the same sources into _build/libfa_sm100_stalltest.so for the
failure-detection GPU test only: every kernel's UMMA issuer waits at pipeline step 1 on an
mbarrier that nothing arrives at, with a 20 ms pipeline-wait limit (teardown waits keep their 2 s
limit), so the kernels' bounded-wait abort path runs on a normal input.  The product library
never contains that wait.
"""
import argparse
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "attention", "libfa_sm100.so")
OPS_OUT = os.path.join(HERE, "attention", "_fa_torch.so")
STALL_OUT = os.path.join(BUILD, "libfa_sm100_stalltest.so")
STALL_FLAGS = ["-DFA_TEST_STALL_STEP=1", "-DFA_WAIT_TIMEOUT_NS=20000000ull"]
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
SOURCES = ["fa_api.cu", "fa_fwd.cu", "fa_bwd.cu", "fa_noalloc.cu", "fa_unfused.cu",
           "fa_rope.cu", "fa_append.cu", "fa_paged.cu", "fa_chunk.cu", "fa_serve_api.cu"]
HEADERS = ["fa_sm100.cuh", "fa_paged.cuh", "fa_softmax.cuh", "fa_internal.h"]

NVCC = os.environ.get("NVCC", "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-I", INCLUDE]


def _newer(src_list, target):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in src_list)


def build(force=False, verbose=False, out=OUT, extra_flags=(), obj_dir=BUILD):
    os.makedirs(obj_dir, exist_ok=True)
    headers = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(INCLUDE, "fa_sm100.h")]
    jobs = []
    objs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(obj_dir, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _newer([s] + headers, o):
            cmd = [NVCC, *ARCH, *FLAGS, *extra_flags, "-c", s, "-o", o]
            if verbose:
                cmd += ["-Xptxas", "-v"]
            jobs.append((src, cmd))

    def run(job):
        name, cmd = job
        r = subprocess.run(cmd, capture_output=True, text=True)
        return name, r

    failed = False
    with ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as ex:
        for name, r in ex.map(run, jobs):
            if r.returncode != 0 or verbose:
                sys.stderr.write(f"--- nvcc {name}\n{r.stdout}{r.stderr}")
            failed |= r.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed")
    if force or jobs or _newer(objs, out):
        cmd = [NVCC, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", out, *objs, "-lcudart_static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return out


def build_ops(force=False, out=OPS_OUT):
    """The native torch binding (see the module docstring); libfa_sm100.so must be built."""
    src = os.path.join(CSRC, "fa_torch.cpp")
    if not force and not _newer([src, os.path.join(INCLUDE, "fa_sm100.h")], out):
        return out
    import torch
    from torch.utils import cpp_extension
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    include = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"], INCLUDE]
    # the C++ runtime is named as a shared library: torch's is, and a second, static one crashes in its streams
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           "-DTORCH_EXTENSION_NAME=_fa_torch", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(x for d in include for x in ("-isystem", d)), src, "-o", out, "-l:libstdc++.so.6", f"-L{os.path.dirname(OUT)}", "-l:libfa_sm100.so",
           "-Wl,-rpath,$ORIGIN", f"-L{lib}", f"-Wl,-rpath,{lib}", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10",
           "-lc10_cuda", "-ltorch_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed")
    return out


def build_stall_test(force=False, verbose=False):
    """The failure-detection test library (see the module docstring)."""
    return build(force, verbose, out=STALL_OUT, extra_flags=STALL_FLAGS,
                 obj_dir=os.path.join(BUILD, "stalltest"))


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
    print(build_ops(force=a.force))
    print(build_stall_test(force=a.force))
