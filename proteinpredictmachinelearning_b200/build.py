"""Builds libppml_b200.so in-tree with nvcc for sm_100a (no JIT cache), and ppml_b200_torch.so, the host side of some of its entries
for torch tensors, with g++ against the installed torch."""
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(OUT_DIR, "libppml_b200.so")
TORCH_BINDING = os.path.join(OUT_DIR, "ppml_b200_torch.so")

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
            raise RuntimeError("nvcc failed: " + " ".join(cmd))

    with ThreadPoolExecutor(max_workers=8) as ex:
        list(ex.map(run, jobs))
    if jobs or not os.path.exists(LIB):
        run([NVCC] + ARCH + ["-shared", "-o", LIB] + objs + ["-Xcompiler", "-fPIC", "-cudart", "static"])
    binding = os.path.join(CSRC, "torch_binding.cpp")
    needs = [binding, os.path.join(HERE, "..", "include", "ppml_b200.h")]
    if force or not os.path.exists(TORCH_BINDING) or any(os.path.getmtime(f) > os.path.getmtime(TORCH_BINDING) for f in needs):
        import torch
        root = os.path.dirname(torch.__file__)
        torch_lib, cuda = os.path.join(root, "lib"), os.path.dirname(os.path.dirname(NVCC))
        include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include"),
                   sysconfig.get_paths()["include"]]
        run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] +
            [f"-isystem{d}" for d in include] +
            [binding, "-o", TORCH_BINDING, "-L" + OUT_DIR, "-l:libppml_b200.so", "-L" + torch_lib, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
             "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
