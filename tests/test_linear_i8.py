"""Linears in 8-bit integers with one scale per token and per output channel: the quantizer against the format's definition
(fp32 quotients, numpy), the product against 64-bit arithmetic.

Bounds.  The integer sums are exact.  Behind them, in fp32: the sum to fp32, times a scale, fused with the second scale and the
bias: three roundings of the product's magnitude and one of the result.  An activation of slope <= 1.13 carries that on
and adds a few units in the last place of its own; the gate and the stored type add one rounding each:
  |error| <= 8 * 2^-24 * (|product| + |bias|) * |gate| + 8 * 2^-24 * |result| + eps(type) / 2 * |result| + smallest step / 2."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from proteinpredictmachinelearning_b200 import PATH_AUTO, PATH_SIMT, PATH_UMMA  # noqa: E402
from proteinpredictmachinelearning_b200 import ops  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def rows(M, K, dtype, seed, pitch=None, shift=0):
    """[M, K] with a given row pitch and start, inside a buffer of its own."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch = pitch or K
    buf = torch.full((M * pitch + shift,), 1e4, device="cuda").to(dtype)
    x = buf[shift:].view(M, pitch)[:, :K]
    x.copy_((torch.randn((M, K), generator=g, device="cuda") * torch.exp(torch.randn(K, generator=g, device="cuda") * 0.5)).to(dtype))
    return x


def ints(M, K, seed, pitch=None, shift=0, low=-128):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch = pitch or (K + 15) // 16 * 16
    buf = torch.full((M * pitch + shift,), 99, device="cuda", dtype=torch.int8)
    q = buf[shift:].view(M, pitch)[:, :K]
    q.copy_(torch.randint(low, 128, (M, K), generator=g, device="cuda", dtype=torch.int32).to(torch.int8))
    return q


def scales(n, seed):
    return torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 0.02 + 1e-3


def quantized(x):
    """The definition in numpy's fp32 (IEEE quotients, round half to even)."""
    x = x.float().cpu().numpy()
    amax = np.abs(x).max(axis=1, initial=0.0)
    with np.errstate(all="ignore"):
        s = np.where(np.isfinite(amax), amax / np.float32(127), np.float32(np.nan)).astype(np.float32)
        q = np.rint(x / s[:, None])
    q = np.where(s[:, None] > 0, q, np.float32(0))
    return np.clip(q, -127, 127).astype(np.int8), s


def act64(y, act):
    return {"none": lambda v: v, "sigmoid": torch.special.expit, "silu": lambda v: v * torch.special.expit(v), "tanh": torch.tanh,
            "relu": lambda v: v.clamp(min=0), "gelu": lambda v: 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v ** 3)))}[act](y)


def check_product(got, A, a_scale, W, w_scale, bias, gate, act):
    prod = (A.double() @ W.double().t()) * a_scale.double()[:, None] * w_scale.double()
    b = torch.zeros_like(w_scale).double() if bias is None else bias.double()
    g = torch.ones((), device="cuda", dtype=torch.float64) if gate is None else gate.double()
    want = act64(prod + b, act) * g
    info = torch.finfo(got.dtype)
    tol = 8 * 2.0 ** -24 * ((prod.abs() + b.abs()) * g.abs() + want.abs()) + info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2
    over = (got.double() - want).abs() > tol
    assert not over.any(), (int(over.sum()), (got.double() - want).abs().max().item())


@pytest.fixture
def no_device_abort():
    yield
    code, where = ops.device_status()
    assert code == 0, f"a kernel gave up a bounded wait: code {code} at site {where:#x}"


# ---- quantizer ---------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,K,pitch,shift", [(1, 1, None, 0), (3, 7, None, 0), (5, 33, 40, 3), (2, 128, None, 0), (9, 256, 512, 0),
                                             (4, 1000, None, 1), (3, 4096, None, 0), (2, 4100, 4104, 0), (1, 20000, None, 0), (700, 96, None, 0)])
def test_quantizer_equals_the_definition(M, K, pitch, shift, dtype):
    x = rows(M, K, dtype, M + K, pitch, shift)
    q, s = ops.quantize_tokens_i8(x)
    wq, ws = quantized(x)
    assert np.array_equal(s.cpu().numpy(), ws)
    assert np.array_equal(q.cpu().numpy(), wq)


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("K", [64, 2048, 12000])
def test_quantizer_ties_zeros_and_extremes(K, dtype):
    """Largest magnitudes at which half steps are representable (ties to even), rows of zeros, negative extremes, the smallest
    and largest finite numbers."""
    x = torch.zeros((8, K), device="cuda")
    n = torch.arange(K, device="cuda", dtype=F32) % 255 - 127
    x[0], x[0, 0] = n * 0.5, 127.0                                    # scale 1: halves
    x[1], x[1, 5] = n, 254.0                                          # scale 2: halves
    x[2], x[2, -1] = n * 0.25, -63.5                                  # scale 0.5, the extreme negative and last
    x[4] = torch.finfo(dtype).smallest_normal * n / 127
    x[5, 3] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps     # the smallest subnormal alone
    x[6], x[6, 1] = 1.0, torch.finfo(dtype).max
    x[7] = -0.0
    x = x.to(dtype)
    q, s = ops.quantize_tokens_i8(x)
    wq, ws = quantized(x)
    assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(q.cpu().numpy(), wq)
    assert not q[3].any() and s[3] == 0


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [5, 70])
def test_rows_with_infinities_or_nan_give_nan_and_leave_the_others(dtype, M, no_device_abort):
    x = rows(M, 272, dtype, 3)
    x[1, 7], x[2, 0], x[4, 271] = float("nan"), float("inf"), float("-inf")
    W, ws = ops.quantize_tokens_i8(rows(40, 272, F32, 4))
    q, s = ops.quantize_tokens_i8(x)
    bad = torch.tensor([i in (1, 2, 4) for i in range(M)], device="cuda")
    assert torch.equal(torch.isnan(s), bad) and not q[bad].any()
    for path in (PATH_AUTO, PATH_SIMT):
        y = ops.linear_i8(x, W, ws, dtype=F32, path=path)
        assert torch.isnan(y[bad]).all()
        check_product(y[~bad], q[~bad], s[~bad], W, ws, None, None, "none")
        few = ops.linear_i8(x[:4], W, ws, dtype=F32, path=path)
        assert torch.isnan(few[1:3]).all() and torch.equal(few[0], y[0]) and torch.equal(few[3], y[3])


@gpu
def test_quantizer_leaves_what_is_behind_a_row():
    x = rows(5, 50, BF16, 1)
    q = torch.full((5, 64), 77, device="cuda", dtype=torch.int8)
    ops.quantize_tokens_i8(x, out=(q[:, :50], torch.empty(5, device="cuda")))
    assert (q[:, 50:] == 77).all()


# ---- product -----------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 16, 8), (1, 1024, 4096), (2, 4096, 256), (3, 100, 5), (4, 64, 33), (7, 272, 130), (8, 2048, 1000), (9, 96, 64), (16, 512, 520),
          (17, 128, 128), (31, 1000, 264), (48, 4096, 512), (64, 144, 2000), (65, 256, 96), (128, 128, 128), (129, 272, 257), (255, 33, 40),
          (257, 640, 512), (408, 128, 128), (700, 1040, 777), (1025, 256, 1032)]


@gpu
@pytest.mark.parametrize("path", [PATH_AUTO, PATH_SIMT])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product_against_64_bits(M, K, N, path, no_device_abort):
    A, W, sa, sw = ints(M, K, 1), ints(N, K, 2), scales(M, 3), scales(N, 4)
    for i, dtype in enumerate((F32, F16, BF16)):
        bias = scales(N, 5) if i != 1 else None
        scale = 1.0 if dtype != F16 else 2.0 ** -6                   # sums of 2^14 * K leave the range of fp16
        check_product(ops.mul_mat_i8(A, sa * scale, W, sw, bias=bias, dtype=dtype, path=path), A, sa * scale, W, sw, bias, None, "none")


@gpu
@pytest.mark.parametrize("M,K,N", [(19001, 144, 96), (40003, 48, 120), (5001, 272, 600), (2600, 1104, 1100), (9000, 2064, 264), (65536, 32, 136),
                                   (1111, 4100, 2056), (300, 128, 20011)])
def test_many_tiles(M, K, N, no_device_abort):
    """More output tiles than SMs, with one and two tiles of channels, one to many steps of K, ragged ends on every side."""
    A, W, sa, sw, bias = ints(M, K, 1), ints(N, K, 2), scales(M, 3), scales(N, 4), scales(N, 5)
    gate = torch.randn((M, N), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    out = torch.full((M + 1, N + 3), -7.0, device="cuda")
    ops.mul_mat_i8(A, sa, W, sw, bias=bias, gate=gate, out=out[:M, :N])
    check_product(out[:M, :N], A, sa, W, sw, bias, gate, "none")
    assert (out[:, N:] == -7).all() and (out[M] == -7).all()
    check_product(ops.mul_mat_i8(A, sa, W, sw, act="silu", dtype=BF16), A, sa, W, sw, None, None, "silu")


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 1024, 256), (5, 80, 40), (24, 512, 264), (140, 64, 96), (300, 256, 520), (33, 100, 41)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu", "gelu", "tanh", "relu"])
def test_epilogue(M, K, N, act, dtype, no_device_abort):
    A, W = ints(M, K, 1), ints(N, K, 2)
    sa, sw, bias = scales(M, 3) * (0.1 / K ** 0.5), scales(N, 4) * 10, scales(N, 5) * 50 - 0.3
    gate = torch.randn((M, N + 8), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").to(dtype)[:, :N]
    out = torch.full((M, N + 16), -7.0, device="cuda", dtype=dtype)
    ops.mul_mat_i8(A, sa, W, sw, bias=bias, gate=gate, act=act, out=out[:, :N])
    check_product(out[:, :N], A, sa, W, sw, bias, gate, act)
    assert (out[:, N:] == -7).all()
    check_product(ops.mul_mat_i8(A, sa, W, sw, act=act, dtype=dtype), A, sa, W, sw, None, None, act)


@gpu
@pytest.mark.parametrize("M,K,N", [(3, 100, 40), (20, 333, 65), (150, 97, 70)])
def test_operands_off_sixteen_bytes(M, K, N, no_device_abort):
    """Pitches and bases that TMA cannot address, an output whose rows are not a multiple of 16 bytes."""
    sa, sw = scales(M, 3), scales(N, 4)
    for pa, ha, pb, hb in ((K, 0, K, 0), (K + 3, 1, K + 1, 0), ((K + 15) // 16 * 16, 4, (K + 15) // 16 * 16, 0), (K + 5, 2, K + 2, 7)):
        A, W = ints(M, K, 1, pa, ha), ints(N, K, 2, pb, hb)
        for dtype in (F32, BF16):
            out = torch.full((M * (N + 1) + 1,), -7.0, device="cuda", dtype=dtype)
            y = out[1:].view(M, N + 1)[:, :N]
            ops.mul_mat_i8(A, sa, W, sw, out=y)
            check_product(y, A, sa, W, sw, None, None, "none")
            assert (out[1:].view(M, N + 1)[:, N] == -7).all() and out[0] == -7


@gpu
def test_tensor_core_path_wants_aligned_operands():
    A, W, s = ints(8, 64, 1, 65), ints(8, 64, 2), scales(8, 3)
    with pytest.raises(RuntimeError, match="status 7"):
        ops.mul_mat_i8(A, s, W, s, path=PATH_UMMA)
    with pytest.raises(RuntimeError, match="status 7"):
        ops.mul_mat_i8(W, s, A, s, path=PATH_UMMA)


@gpu
@pytest.mark.parametrize("M,N", [(1, 5), (6, 40), (40, 24), (200, 130)])
def test_largest_sums_are_exact(M, N, no_device_abort):
    """K at its limit with every product at its largest: 128 * 128 * 131071 is just inside int32."""
    K = 131071
    A, W = torch.full((M, 131072), -128, device="cuda", dtype=torch.int8)[:, :K], torch.full((N, 131072), -128, device="cuda", dtype=torch.int8)[:, :K]
    W[1:].neg_()                                                      # -128 stays -128
    W[2:].fill_(127)
    s, one = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    for path in (PATH_AUTO, PATH_SIMT):
        y = ops.mul_mat_i8(A, s, W, one, path=path)
        assert (y[:, :2] == float(128 * 128 * K)).all()               # 2147467264 is a multiple of 128: fp32 holds it
        assert (y[:, 2:].double() - (-128.0 * 127 * K)).abs().max() <= 2.0 ** 31 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 65, 130, 1000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_is_quantizer_and_product(M, dtype, no_device_abort):
    """One call, two calls, the CUDA-core path and any part of the tokens give the same bits."""
    for K, N in ((272, 200), (100, 64), (2049, 72), (528, 3500), (144, 9000), (5000, 9), (8192, 24), (8193, 24)):
        x = rows(M, K, dtype, M, K + 8)
        W, ws = ops.quantize_tokens_i8(rows(N, K, F32, 9) * 0.02)
        bias = scales(N, 5)
        q, s = ops.quantize_tokens_i8(x)
        y = ops.linear_i8(x, W, ws, bias=bias)
        assert y.dtype == dtype
        check_product(y, q, s, W, ws, bias, None, "none")
        assert torch.equal(y, ops.mul_mat_i8(q, s, W, ws, bias=bias, dtype=dtype))
        assert torch.equal(y, ops.linear_i8(x, W, ws, bias=bias, path=PATH_SIMT))
        assert torch.equal(y[M // 2:], ops.linear_i8(x[M // 2:], W, ws, bias=bias))
    x, W = rows(M, 272, dtype, 1, 275, 3), ints(90, 272, 2, 273, 1)           # nothing on 16 bytes
    gate = rows(M, 90, F32, 4)
    y = ops.linear_i8(x, W, scales(90, 2), gate=gate, act="gelu", dtype=F32)
    q, s = ops.quantize_tokens_i8(x)
    check_product(y, q, s, W, scales(90, 2), None, gate, "gelu")


@gpu
@pytest.mark.parametrize("M", [5, 7, 8, 15, 23, 25, 32, 40, 41, 56, 63, 72, 95, 97, 104, 120, 127, 136, 161, 192, 200, 223, 225, 239, 256, 257, 450])
@pytest.mark.parametrize("act,K", [("silu", 64), ("relu", 64), ("none", 64), ("sigmoid", 1024)])
def test_every_share_of_a_tile(M, act, K, no_device_abort):
    """Tiles whose tokens fall unevenly to the warps of the epilogue, rows on and off the width of a paired store."""
    A, W = ints(M, K, 1), ints(256, K, 2)
    sa, sw = scales(M, 3) * (0.1 / K ** 0.5), scales(256, 4) * 10
    for N, dtype, pitch in ((256, BF16, 256), (130, F16, 133), (256, F32, 257)):
        gate = rows(M, N, dtype, 5)
        out = torch.full((M + 1, pitch), -7.0, device="cuda", dtype=dtype)
        for g in (None, gate):
            ops.mul_mat_i8(A, sa, W[:N], sw[:N], gate=g, act=act, out=out[:M, :N])
            check_product(out[:M, :N], A, sa, W[:N], sw[:N], None, g, act)
        assert (out[M] == -7).all() and (out[:, N:] == -7).all()


@gpu
@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("K", [1, 15, 17, 496, 511, 513, 1024, 1025, 1536, 2047, 2048])
def test_few_tokens_at_the_ends_of_a_step(M, K, no_device_abort):
    for N, pitch, shift in ((1, None, 0), (15, None, 0), (2367, None, 0), (2385, None, 0), (4741, None, 0), (100, K + 1, 3)):
        x, W, ws, bias = rows(M, K, BF16, M, K + 3, 1), ints(N, K, 2, pitch, shift), scales(N, 3), scales(N, 4)
        q, s = ops.quantize_tokens_i8(x)
        out = torch.full((M + 1, N + 1), -7.0, device="cuda")
        ops.linear_i8(x, W, ws, bias=bias, out=out[:M, :N])
        assert torch.equal(out[:M, :N], ops.mul_mat_i8(q, s, W, ws, bias=bias, path=PATH_SIMT))
        assert (out[M] == -7).all() and (out[:, N] == -7).all()


@gpu
@pytest.mark.parametrize("M,K,N", [(2, 272, 200), (30, 2048, 136), (300, 272, 264), (9000, 80, 300)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gate_may_be_the_output(M, K, N, dtype, no_device_abort):
    x, gate = rows(M, K, dtype, 1), rows(M, N, dtype, 2)
    W, ws = ops.quantize_tokens_i8(rows(N, K, F32, 3) * 0.02)
    for path in (PATH_AUTO, PATH_SIMT):
        want = ops.linear_i8(x, W, ws, gate=gate, act="silu", path=path)
        own = gate.clone()
        ops.linear_i8(x, W, ws, gate=own, act="silu", out=own, path=path)
        assert torch.equal(own, want)


@gpu
def test_empty_batches():
    W, ws = ints(8, 64, 1), scales(8, 2)
    x = torch.empty((0, 64), device="cuda")
    q, s = ops.quantize_tokens_i8(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    assert ops.mul_mat_i8(q, s, W, ws).shape == (0, 8) and ops.linear_i8(x, W, ws).shape == (0, 8)


@gpu
def test_offsets_beyond_32_bits(no_device_abort):
    """Rows that start beyond 2^31 elements, of the input, the integers and the output."""
    K, N, pitch = 64, 40, (1 << 31) // 3 // 16 * 16
    buf = torch.empty(4 * pitch + 64, device="cuda", dtype=torch.int8)
    A = torch.as_strided(buf, (5, K), (pitch, 1))
    A.copy_(ints(5, K, 1))
    W, sa, sw = ints(N, K, 2), scales(5, 3), scales(N, 4)
    wide = torch.empty(4 * pitch + 64, device="cuda", dtype=BF16)
    y = torch.as_strided(wide, (5, N), (pitch, 1))
    for path in (PATH_AUTO, PATH_SIMT):
        y.zero_()
        ops.mul_mat_i8(A, sa, W, sw, out=y, path=path)
        check_product(y, A, sa, W, sw, None, None, "none")
    x = torch.as_strided(wide, (5, K), (pitch, 1))
    x.copy_(rows(5, K, BF16, 8))
    q, s = ops.quantize_tokens_i8(x)
    wq, wsc = quantized(x)
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), wsc)
    check_product(ops.linear_i8(x, W, sw, dtype=F32), q, s, W, sw, None, None, "none")


@gpu
@pytest.mark.parametrize("M", [1, 20, 300])
def test_captured_calls_replay_on_new_inputs(M, no_device_abort):
    """Two graphs of the same call alive at once, replayed in turn and on another stream than they were captured on."""
    K, N = 272, 136
    W, ws = ops.quantize_tokens_i8(rows(N, K, F32, 9))
    x = [rows(M, K, BF16, i) for i in (1, 2)]
    graphs, outs = [], []
    ops.linear_i8(x[0], W, ws)
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.linear_i8(x[i], W, ws, act="silu"))
        graphs.append(g)
    for r in range(3):
        for i in range(2):
            x[i].copy_(rows(M, K, BF16, 10 + 2 * r + i))
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in (1, 0):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], ops.linear_i8(x[i], W, ws, act="silu"))


@gpu
def test_two_streams_at_once(no_device_abort):
    """Calls of both sizes on two streams without a wait between them."""
    W, ws = ops.quantize_tokens_i8(rows(264, 512, F32, 9))
    xs = [rows(m, 512, BF16, m) for m in (1, 700, 40, 900)]
    want = [ops.linear_i8(x, W, ws) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = {}
    for r in range(4):
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[(i + r) % 2]):
                got[r, i] = ops.linear_i8(x, W, ws)
    torch.cuda.synchronize()
    for (r, i), y in got.items():
        assert torch.equal(y, want[i]), (r, i)


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_bad_arguments_are_refused_on_the_host(lib):
    p = C.c_void_p(64)
    quant = lambda *a: lib.ppml_b200_quantize_tokens_i8(*a, None)     # noqa: E731
    assert quant(p, 0, 8, p, 8, p, -1, 8) == 1 and quant(p, 0, 8, p, 8, p, 4, 0) == 1
    assert quant(p, 3, 8, p, 8, p, 4, 8) == 1 and quant(p, -1, 8, p, 8, p, 4, 8) == 1
    assert quant(p, 0, 7, p, 8, p, 4, 8) == 1 and quant(p, 0, 8, p, 7, p, 4, 8) == 1
    assert quant(None, 0, 8, p, 8, p, 4, 8) == 1 and quant(p, 0, 8, None, 8, p, 4, 8) == 1 and quant(p, 0, 8, p, 8, None, 4, 8) == 1
    assert quant(C.c_void_p(66), 0, 8, p, 8, p, 4, 8) == 1 and quant(C.c_void_p(65), 2, 8, p, 8, p, 4, 8) == 1
    assert quant(p, 0, 8, p, 8, p, 1 << 31, 8) == 1
    assert quant(None, 0, 8, None, 8, None, 0, 8) == 0                # no tokens, no work

    names = ("A", "lda", "a_scale", "B", "ldb", "b_scale", "C", "ldc", "c_type", "M", "K", "N", "bias", "gate", "ld_gate", "act", "path")
    good = (p, 16, p, p, 16, p, p, 8, 0, 4, 16, 8, None, None, 0, 0, 0)

    def mm(**kw):
        return lib.ppml_b200_mul_mat_i8(*[kw.get(n, v) for n, v in zip(names, good)], None)
    for bad in (dict(M=-1), dict(K=0), dict(N=0), dict(K=17), dict(lda=15), dict(ldb=15), dict(ldc=7), dict(c_type=3), dict(act=6), dict(act=-1),
                dict(path=3), dict(A=None), dict(B=None), dict(C=None), dict(a_scale=None), dict(b_scale=None), dict(gate=p, ld_gate=7),
                dict(C=C.c_void_p(66)), dict(C=C.c_void_p(65), c_type=1), dict(bias=C.c_void_p(66)), dict(a_scale=C.c_void_p(65))):
        assert mm(**bad) == 1, bad
    assert mm(K=131072, lda=1 << 18, ldb=1 << 18) == 9
    assert mm(N=4194241, ldc=4194241, path=1) == 9
    assert mm(M=0) == 0 and mm(M=0, A=None, C=None, a_scale=None) == 0
    assert mm(path=2, A=C.c_void_p(68)) == 7 and mm(path=2, lda=17) == 7 and mm(path=2, B=C.c_void_p(72)) == 7 and mm(path=2, ldb=24) == 7

    assert lib.ppml_b200_linear_i8_workspace(5, 17) == 5 * 32 + 32 and lib.ppml_b200_linear_i8_workspace(0, 17) == 0
    assert lib.ppml_b200_linear_i8_workspace(4, 2048) == 0 and lib.ppml_b200_linear_i8_workspace(4, 2049) == 4 * 2064 + 16
    assert lib.ppml_b200_linear_i8_workspace(1, 8192) == 0 and lib.ppml_b200_linear_i8_workspace(2, 4097) == 2 * 4112 + 16
    names = ("X", "x_type", "ld_x", "B", "ldb", "b_scale", "C", "ldc", "c_type", "M", "K", "N", "bias", "gate", "ld_gate", "act", "path", "ws", "bytes")
    good = (p, 0, 16, p, 16, p, p, 8, 0, 6, 16, 8, None, None, 0, 0, 0, p, 128)

    def lin(**kw):
        return lib.ppml_b200_linear_i8(*[kw.get(n, v) for n, v in zip(names, good)], None)
    for bad in (dict(X=None), dict(x_type=3), dict(ld_x=15), dict(X=C.c_void_p(66)), dict(B=None), dict(N=0), dict(act=9)):
        assert lin(**bad) == 1, bad
    assert lin(ws=None) == 3 and lin(bytes=127) == 3 and lin(M=4, path=2) == 7 and lin(ws=C.c_void_p(72)) == 3
    assert lin(M=0, ws=None, bytes=0) == 0 and lin(K=131072, ldb=1 << 18, ld_x=1 << 18) == 9


@gpu
def test_wrong_tensors_are_refused():
    x, W, ws = rows(4, 32, BF16, 1), ints(8, 32, 2), scales(8, 3)
    q, s = ops.quantize_tokens_i8(x)
    for bad in (lambda: ops.quantize_tokens_i8(x.to(torch.int32)), lambda: ops.quantize_tokens_i8(x.cpu()), lambda: ops.quantize_tokens_i8(x[0]),
                lambda: ops.quantize_tokens_i8(x.t()), lambda: ops.quantize_tokens_i8(x, out=(q[:, :16], s)),
                lambda: ops.quantize_tokens_i8(x, out=(q, s.double())), lambda: ops.mul_mat_i8(q.float(), s, W, ws),
                lambda: ops.mul_mat_i8(q, s, W[:, :16], ws), lambda: ops.mul_mat_i8(q, s[:3], W, ws), lambda: ops.mul_mat_i8(q, s, W, ws[:7]),
                lambda: ops.mul_mat_i8(q, s, W.cpu(), ws), lambda: ops.mul_mat_i8(q, s, W, ws, bias=ws.half()),
                lambda: ops.mul_mat_i8(q, s, W, ws, gate=torch.zeros((4, 8), device="cuda"), dtype=BF16),
                lambda: ops.mul_mat_i8(q, s, W, ws, act="swish"), lambda: ops.mul_mat_i8(q, s, W, ws, dtype=torch.float64),
                lambda: ops.mul_mat_i8(q, s, W, ws, out=torch.zeros((8, 4), device="cuda").t()),
                lambda: ops.mul_mat_i8(q, s, W, ws, out=torch.zeros((1, 8), device="cuda").expand(4, 8)),
                lambda: ops.linear_i8(x, W, None), lambda: ops.linear_i8(x, W, ws, path="auto"), lambda: ops.linear_i8(x, W, ws, dtype="bf16"),
                lambda: ops.linear_i8(x, W[:, ::2], ws), lambda: ops.linear_i8(x[:, ::2], W[:, :16], ws), lambda: ops.linear_i8(x, W, ws, dtype=torch.int8)):
        with pytest.raises(ValueError):
            bad()
