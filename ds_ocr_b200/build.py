"""Builds the in-tree CUDA library ds_ocr_b200/libds_cuda.so for sm_100a.

nvcc compiles every .cu under csrc/ (plus the host C file synth.c) with
-gencode arch=compute_100a,code=sm_100a into one shared library exporting the
C ABI of include/ds_cuda.h. Runs without a GPU (cross-compilation). Where
torch with CUDA is installed, g++ then builds the module ds_ocr_b200._spec
(csrc/spec_torch.cpp), the speculative-decoding calls on torch tensors.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libds_cuda.so")
SPEC = os.path.join(HERE, "_spec.so")
BUILD = os.path.join(ROOT, "_build")
SPEC_FOR = os.path.join(BUILD, "_spec.for")  # the torch and Python that SPEC was built for

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc():
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "nvcc"


def sources():
    cu = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))
    return [os.path.join(CSRC, f) for f in cu]


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose=False, force=False):
    os.makedirs(BUILD, exist_ok=True)
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hdrs.append(os.path.join(ROOT, "include", "ds_cuda.h"))
    objs = []
    procs = []
    for src in sources():
        obj = os.path.join(BUILD, os.path.basename(src) + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + hdrs):
            cmd = [_nvcc(), *NVCC_FLAGS, "-I", CSRC, "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd))
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    synth_o = os.path.join(BUILD, "synth.c.o")
    synth_c = os.path.join(CSRC, "synth.c")
    if force or _stale(synth_o, [synth_c]):
        procs.append((synth_c, subprocess.Popen(
            ["gcc", "-O2", "-fPIC", "-c", synth_c, "-o", synth_o],
            stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append((src, out.decode(errors="replace")))
        elif verbose and out:
            print(out.decode(errors="replace"))
    if failed:
        for src, out in failed:
            sys.stderr.write(f"--- {src}\n{out}\n")
        raise RuntimeError("nvcc failed for: " + ", ".join(s for s, _ in failed))
    objs.append(synth_o)
    if force or _stale(LIB, objs):
        cmd = [_nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB, *objs,
               "-lcudart", "-lcuda", "-lpthread", "-ldl", "-lm"]
        if verbose:
            print(" ".join(cmd))
        subprocess.check_call(cmd)
    try:
        build_spec(verbose, force)
    except (OSError, subprocess.CalledProcessError) as e:  # the library stands without it; its first use says why again
        print(f"{SPEC} not built: {e}", file=sys.stderr)
    return LIB


def _read(path):
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return None


def _write(path, text):
    os.makedirs(os.path.dirname(path), exist_ok=True)
    with open(path, "w") as f:
        f.write(text)


def _spec_abi():
    """What the torch module depends on beside its sources."""
    import sysconfig
    import torch
    return f"torch {torch.__version__} cuda {torch.version.cuda} {sysconfig.get_config_var('SOABI')}"


def spec_is_for_another():
    """Whether the torch module was built for another torch or Python."""
    return _read(SPEC_FOR) not in (None, _spec_abi())


def build_spec(verbose=False, force=False):
    """The torch module _spec.so (it is given the C ABI's addresses, not linked
    to the library: DS_CUDA_LIB may name another one)."""
    try:
        import torch
    except ImportError:
        return None
    if torch.version.cuda is None:
        return None
    import sysconfig
    src = os.path.join(CSRC, "spec_torch.cpp")
    if not (force or _read(SPEC_FOR) != _spec_abi() or _stale(SPEC, [src, os.path.join(ROOT, "include", "ds_cuda.h")])):
        return SPEC
    base = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())) or "/usr/local/cuda", "include")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", src, "-o", SPEC,
           "-I", os.path.join(ROOT, "include"), "-isystem", sysconfig.get_paths()["include"],
           "-isystem", os.path.join(base, "include"),
           "-isystem", os.path.join(base, "include", "torch", "csrc", "api", "include"), "-isystem", cuda,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-L", os.path.join(base, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd))
    if os.path.exists(SPEC):  # (an old one with other structs must not stay where this fails)
        os.remove(SPEC)
    subprocess.check_call(cmd)
    _write(SPEC_FOR, _spec_abi())
    return SPEC


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, force="-f" in sys.argv)
    print(LIB)
