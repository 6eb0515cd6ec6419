"""Linears in 8-bit integers at the edges: results that share memory with the input, activations over their whole range,
results that no memory holds."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from proteinpredictmachinelearning_b200 import PATH_AUTO, PATH_SIMT, PATH_UMMA  # noqa: E402
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


# ---- activations over their whole range --------------------------------------------------------------------------------
U = 2.0 ** -24


def act_of(v, act):
    """The value, and the argument of its sigmoid, in 64 bits."""
    v = v.double()
    s = v if act != "gelu" else 2 * 0.7978845608028654 * (v + 0.044715 * v ** 3)
    return (1 if act == "sigmoid" else v) / (1 + torch.exp(-s)), s


def reach(act, lowest):
    """Arguments on either side whose sigmoid takes arguments from `lowest` to 200."""
    v = torch.cat((torch.linspace(lowest, 12, 20001, device="cuda"), torch.linspace(12, 200, 501, device="cuda"), 10.0 ** torch.linspace(-30, 0, 61, device="cuda"),
                   -(10.0 ** torch.linspace(-30, 0, 61, device="cuda"))))
    if act == "gelu":
        v = v.clamp(-20, 20)
    return v[act_of(v, act)[1] >= lowest]


@gpu
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("path,lowest,slope", [(PATH_SIMT, -88.5, 0), (PATH_UMMA, -87.0, 2), (PATH_AUTO, -87.0, 2)])
def test_activations_of_the_product(act, path, lowest, slope):
    """One integer 1 on either side: the token's scale goes into the activation as it is.  expf is off by 2 units in the last place
    (4 u), the sum and the division by u each; the hardware's functions as the header says; GELU's argument has seven
    roundings of itself.  What is below the smallest normal number may be off by a step there."""
    v = reach(act, lowest)
    A, W = torch.ones((v.numel(), 16), device="cuda", dtype=torch.int8)[:, :1], torch.ones((3, 16), device="cuda", dtype=torch.int8)[:, :1]
    want, s = act_of(v, act)
    tol = (8 + (8 if act == "gelu" else slope) * s.abs()) * U * want.abs() + (2.0 ** -126 if slope else 2.0 ** -148)
    y = ops.mul_mat_i8(A, v, W, torch.ones(3, device="cuda"), act=act, path=path)
    assert ((y.double() - want[:, None]).abs() <= tol[:, None]).all(), ((y.double() - want[:, None]).abs() / tol[:, None]).max()


@gpu
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("path,lowest,slope", [(PATH_SIMT, -88.5, 0), (PATH_AUTO, -87.0, 2)])
def test_activations_of_a_few_tokens(act, path, lowest, slope):
    """The one kernel for a few tokens: its bias goes into the activation as it is, behind a token of zeros."""
    v = reach(act, lowest)
    W, ws = torch.ones((v.numel(), 16), device="cuda", dtype=torch.int8), torch.ones(v.numel(), device="cuda")
    want, s = act_of(v, act)
    tol = (8 + (8 if act == "gelu" else slope) * s.abs()) * U * want.abs() + (2.0 ** -126 if slope else 2.0 ** -148)
    y = ops.linear_i8(torch.zeros((3, 16), device="cuda"), W, ws, bias=v, act=act, path=path)
    assert ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() / tol).max()


# ---- memory ------------------------------------------------------------------------------------------------------------
@gpu
def test_a_result_that_no_memory_holds():
    """4 TB: the allocator's own error, as from any torch call, and the next call runs."""
    x, W, ws = rand((1 << 20, 16), 1), torch.ones((1 << 20, 16), device="cuda", dtype=torch.int8), torch.ones(1 << 20, device="cuda")
    with pytest.raises(torch.OutOfMemoryError):
        ops.linear_i8(x, W, ws)
    assert torch.equal(ops.linear_i8(x[:8], W[:8], ws[:8]), ops.linear_i8(x, W[:8], ws[:8])[:8])
