"""Linears in 8-bit integers at the edges: results that share memory with the input, activations over their whole range,
results that no memory holds, and every cut of the product into tiles."""
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


# ---- one of two results given ------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("M,K", [(3, 64), (40, 1000)])
def test_quantizer_writes_into_what_it_is_given(M, K):
    x = rand((M, K), 1, BF16)
    q, s = ops.quantize_tokens_i8(x)
    for give_q, give_s in ((True, True), (True, False), (False, True)):
        mine = (torch.full((M, K), 77, device="cuda", dtype=torch.int8) if give_q else None, torch.full((M,), -7.0, device="cuda") if give_s else None)
        got = ops.quantize_tokens_i8(x, out=mine)
        assert torch.equal(got[0], q) and torch.equal(got[1], s)
        assert all(m is None or m is t for m, t in zip(mine, got))


# ---- every cut of the product ------------------------------------------------------------------------------------------
# Sizes at which the choice falls on each kind of tile, with ends of tiles of every length (tokens of a tile: sizes).
PARTS = {  # clusters of two, four and eight CTAs that share a tile's K
    "16": [(5, 1185, 4352), (5, 917, 40), (5, 2090, 40)],
    "32": [(20, 2048, 8192), (1145, 1159, 43), (35, 994, 41), (18, 938, 40), (33, 1932, 41), (17, 2087, 40)],
    "48": [(48, 4096, 8192), (35, 1697, 5142), (34, 1206, 2082), (33, 1928, 935)],
    "64": [(200, 8192, 1024), (3459, 2462, 41), (3195, 2435, 46), (1287, 1823, 41), (1136, 1916, 41), (586, 3796, 45), (491, 3651, 42)],
    "80": [(66, 3216, 5164), (69, 1862, 3250), (65, 2074, 1620)],
    "96": [(4813, 2651, 52), (5246, 3079, 42), (2406, 2501, 49), (2955, 2239, 43), (1183, 2746, 43), (1141, 2563, 50)],
    "112": [(100, 4987, 4769), (98, 2506, 2836), (105, 4885, 1047)],
    "128": [(7819, 3988, 41), (7295, 4061, 52), (3207, 4032, 40), (3784, 3985, 40), (1537, 7849, 74), (1622, 7769, 41), (1649, 8249, 52)]}
SINGLE = {  # one CTA a tile
    "64": [(5005, 18, 40), (4833, 17, 46)], "96": [(10289, 16, 40), (9758, 17, 40), (9790, 16, 42)],
    "128": [(14729, 16, 47), (15803, 16, 42), (15452, 16, 48), (14712, 16, 45)],
    "160": [(22579, 21, 45), (22463, 19, 44), (20249, 17, 42), (20313, 16, 41)],
    "192": [(8191, 64, 300), (27845, 16, 40), (24615, 18, 41), (24079, 18, 41), (26629, 16, 40), (23798, 16, 54)],
    "224": [(10000, 64, 300), (30047, 20, 42), (30541, 17, 45), (28802, 18, 41), (30179, 16, 46), (28668, 20, 49)],
    "256": [(5000, 64, 777), (34313, 16, 43), (34352, 18, 55), (36176, 23, 40), (35183, 16, 42), (36760, 16, 44), (33972, 17, 51), (33236, 17, 52),
            (34807, 16, 75)]}
PAIRS = {  # two CTAs a tile of 256 channels
    "64": [(2589, 1412, 152), (2609, 1487, 136)], "96": [(4923, 948, 138), (4843, 986, 129), (5454, 961, 130)],
    "128": [(7321, 738, 145), (7131, 757, 141), (7535, 682, 138)], "160": [(11364, 516, 129), (10809, 600, 131), (11196, 522, 154)],
    "192": [(12700, 431, 165), (11991, 387, 130), (13428, 387, 135)], "224": [(15908, 505, 157), (15049, 408, 130), (15384, 443, 134), (16329, 419, 145)],
    "256": [(17409, 258, 157), (16674, 265, 156), (16986, 308, 129), (16745, 257, 135), (18312, 266, 150), (16828, 289, 152), (450, 263, 6672),
            (17893, 258, 167)]}


def check(got, want, tol):
    """NaN fails, in what is wanted too."""
    assert torch.isfinite(want).all()
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (int((~(off <= tol)).sum()), off.max().item())


@pytest.fixture
def no_device_abort():
    yield
    code, where = ops.device_status()
    assert code == 0, f"a kernel gave up a bounded wait: code {code} at site {where:#x}"


@gpu
@pytest.mark.parametrize("kind,sizes", [(f"{k}-{t}", s) for k, d in (("parts", PARTS), ("single", SINGLE), ("pairs", PAIRS)) for t, s in d.items()],
                         ids=lambda v: v if isinstance(v, str) else "")
def test_every_cut(kind, sizes, no_device_abort):
    """Each type with nothing, an activation, a gate, and both behind the sum, rows that lie close and rows that lie apart, against 64
    bits.  The integer sum is exact; its conversion, two factors and the sum with the bias are 4 roundings of |product| + |bias|, which
    an activation of slope 1.13 at most carries on; its own bound is (8 + 8 |v|) u of the result at worst, with |result| <= |v| and |v|
    below 10 here; the gate and the stored type round once more each."""
    for M, K, N in sizes:
        g = torch.Generator(device="cuda").manual_seed(M + K + N)
        draw = lambda *shape: torch.randn(shape, generator=g, device="cuda")     # noqa: E731
        A, W = ((draw(n, (K + 15) // 16 * 16) * 40).round().clamp(-128, 127).to(torch.int8)[:, :K] for n in (M, N))
        sa, sw, bias = draw(M).abs().clamp(0.1, 2) / (1600 * K ** 0.5), draw(N).abs().clamp(0.1, 2), draw(N)
        prod = (A.double() @ W.double().t()) * sa.double()[:, None] * sw.double()
        for dtype in (F32, F16, BF16):
            half = torch.finfo(dtype).eps / 2
            gate = draw(M, N + 2).to(dtype)[:, 1:N + 1]
            for act, b, h, pitch in (("none", bias, None, N), ("none", None, gate, N + 3), ("silu", bias, None, (N + 1) // 2 * 2), ("silu", None, gate, N),
                                     ("gelu", bias, gate, N + 5)):
                x = prod if b is None else prod + b.double()
                size = prod.abs() + (0 if b is None else b.double().abs())
                v = x if act != "gelu" else 2 * 0.7978845608028654 * (x + 0.044715 * x ** 3)
                want = x if act == "none" else x / (1 + torch.exp(-v))
                tol = 1.13 * 4 * U * size + (0 if act == "none" else (8 + 8 * v.abs()) * U * want.abs())
                if h is not None:
                    want, tol = want * h.double(), tol * h.double().abs() + U * (want * h.double()).abs()
                tol = tol * (1 + half) + half * want.abs() + torch.finfo(dtype).smallest_normal * half
                out = torch.full((M + 1, pitch), -7.0, device="cuda", dtype=dtype)
                ops.mul_mat_i8(A, sa, W, sw, bias=b, gate=h, act=act, out=out[:M, :N])
                check(out[:M, :N], want, tol)
                assert (out[M] == -7).all() and (out[:, N:] == -7).all()
