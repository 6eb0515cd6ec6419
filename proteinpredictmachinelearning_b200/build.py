"""Builds libppml_b200.so in-tree with nvcc for sm_100a (no JIT cache), and, where a torch with CUDA is installed, ppml_b200_torch.so,
the host side of some of its entries for torch tensors, with g++ against that torch."""
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(OUT_DIR, "libppml_b200.so")
TORCH_BINDING = os.path.join(OUT_DIR, "ppml_b200_torch.so")
TORCH_STAMP = os.path.join(OUT_DIR, "ppml_b200_torch.txt")      # the torch and the Python that the binding was built against

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=default"]

SOURCES = ["simt_kernels.cu", "simt_contract.cu", "umma_gemm.cu", "umma_q8.cu", "umma_attn.cu", "attn_exact.cu", "attn_backward.cu", "attn_backward_short.cu", "attn_mma8.cu", "noalloc.cu", "peer_exchange.cu", "i8_simt.cu", "i8_few.cu", "umma_i8.cu", "qk_norm_rope.cu", "capi.cu",
           "tma_host.cpp", "host_quant.cpp", "q8_file.cpp", "ppml_forwarders.cpp"]


def _sources():
    return [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]


def _stale(obj, src):
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    deps = [src] + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh", ".inc"))]
    deps.append(os.path.join(HERE, "..", "include", "ppml_b200.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _cuda_root():
    """The directory above nvcc's `bin`, or else one of the usual ones, that holds CUDA's headers."""
    roots = [os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(NVCC) or NVCC))), os.environ.get("CUDA_HOME"), "/usr/local/cuda"]
    return next((r for r in roots if r and os.path.exists(os.path.join(r, "include", "cuda_runtime.h"))), roots[0])


def _installed_torch():
    """Name of the installed torch and of this Python; None without torch."""
    if importlib.util.find_spec("torch") is None:
        return None
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        import torch
        version = torch.__version__
    return f"torch {version}, {sys.implementation.cache_tag}"


def _binding_stale(installed):
    if not os.path.exists(TORCH_BINDING) or not os.path.exists(TORCH_STAMP):
        return True
    with open(TORCH_STAMP) as f:
        if f.read() != installed:
            return True
    needs = [os.path.join(CSRC, "torch_binding.cpp"), os.path.join(HERE, "..", "include", "ppml_b200.h")]
    return any(os.path.getmtime(f) > os.path.getmtime(TORCH_BINDING) for f in needs)


def build_torch_binding(run, force=False):
    """The library does not need it: without a torch that has CUDA it is left out, with a line on stderr."""
    installed = _installed_torch()
    if installed is None:
        sys.stderr.write("torch is not installed: ppml_b200_torch.so is not built (the C ABI does not need it)\n")
        return
    if not force and not _binding_stale(installed):
        return
    import torch
    if torch.version.cuda is None:
        sys.stderr.write("the installed torch has no CUDA: ppml_b200_torch.so is not built (the C ABI does not need it)\n")
        return
    root = os.path.dirname(torch.__file__)
    torch_lib = os.path.join(root, "lib")
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), os.path.join(_cuda_root(), "include"),
               sysconfig.get_paths()["include"]]
    run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
         f'-DPPML_TORCH_VERSION="{torch.__version__}"'] +
        [f"-isystem{d}" for d in include] +
        [os.path.join(CSRC, "torch_binding.cpp"), "-o", TORCH_BINDING, "-L" + OUT_DIR, "-l:libppml_b200.so", "-L" + torch_lib, "-ltorch_python", "-ltorch",
         "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"])
    with open(TORCH_STAMP, "w") as f:
        f.write(installed)


def build(force=False, verbose=False):
    os.makedirs(os.path.join(OUT_DIR, "obj"), exist_ok=True)
    objs, jobs = [], []
    for s in _sources():
        src = os.path.join(CSRC, s)
        obj = os.path.join(OUT_DIR, "obj", os.path.splitext(s)[0] + ".o")
        objs.append(obj)
        if force or _stale(obj, src):
            cmd = [NVCC] + ARCH + COMMON + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0 or verbose:
            sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        if r.returncode != 0:
            raise RuntimeError(os.path.basename(cmd[0]) + " failed: " + " ".join(cmd))

    with ThreadPoolExecutor(max_workers=8) as ex:
        list(ex.map(run, jobs))
    if jobs or not os.path.exists(LIB):
        run([NVCC] + ARCH + ["-shared", "-o", LIB] + objs + ["-Xcompiler", "-fPIC", "-cudart", "static"])
    build_torch_binding(run, force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
