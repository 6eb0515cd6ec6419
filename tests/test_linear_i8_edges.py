"""Linears in 8-bit integers at the edges: results that share memory with the input."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from proteinpredictmachinelearning_b200 import PATH_AUTO, PATH_SIMT  # noqa: E402
from proteinpredictmachinelearning_b200 import ops  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def rand(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


# ---- a result that shares memory with the input ------------------------------------------------------------------------
def test_one_kernel_refuses_a_result_over_its_input(lib):
    """The one kernel for a few tokens reads X until its end.  Host side only: every call here is refused."""
    p = C.c_void_p(4096)

    def linear(M, ld_x, ldc, at_c, x_type=0, c_type=0, K=16, N=8):
        return lib.ppml_b200_linear_i8(p, x_type, ld_x, p, K, p, C.c_void_p(at_c), ldc, c_type, M, K, N, None, None, 0, 0, 0, None, 0, None)
    assert linear(1, 16, 8, 4096) == 1 and linear(4, 16, 16, 4096) == 1
    assert linear(1, 16, 8, 4096 + 60) == 1 and linear(1, 16, 8, 4096 - 28) == 1       # the last element of either
    assert linear(1, 16, 8, 4096 + 30, 1, 1) == 1 and linear(1, 16, 8, 4096 - 14, 2, 2) == 1
    assert linear(3, 24, 24, 4096 + 24 * 4 * 2 + 60) == 1                               # the last row of x alone
    assert linear(3, 40, 40, 4096 + 60) == 1 and linear(4, 24, 8, 4096 + 64) == 1       # pitches of its own: a later row


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,K", [(1, 8192), (2, 4096), (3, 2048), (4, 2048), (4, 100), (5, 512), (300, 272)])
def test_result_may_share_memory_with_the_input(M, K, dtype):
    """In place, one row or a few columns further on, and beside the input in the same rows."""
    W, ws = ops.quantize_tokens_i8(rand((K, K), 1) * 0.05)
    bias, x = rand((K,), 2), rand((M, K), 3, dtype)
    for path in (PATH_AUTO, PATH_SIMT):
        want = ops.linear_i8(x, W, ws, bias=bias, path=path)
        mine = x.clone()
        assert ops.linear_i8(mine, W, ws, bias=bias, path=path, out=mine) is mine and torch.equal(mine, want)
        for shift in (8, K, -8):
            buf = torch.zeros(M * K + K + 16, device="cuda", dtype=dtype)
            a, b = (buf[8 + s:8 + s + M * K].view(M, K) for s in (0, shift))
            a.copy_(x)
            assert torch.equal(ops.linear_i8(a, W, ws, bias=bias, path=path, out=b), want)
        buf = torch.zeros((M, 2 * K + 8), device="cuda", dtype=dtype)
        buf[:, :K] = x
        assert torch.equal(ops.linear_i8(buf[:, :K], W, ws, bias=bias, path=path, out=buf[:, K + 8:]), want)
        assert torch.equal(buf[:, :K], x) and not buf[:, K:K + 8].any()
