"""Norms of queries and keys for each head with the position rotation, forward and backward, against 64-bit arithmetic; and the
path they stand in: 8-bit projection, norm and rotation, attention, attention backward.

Bounds (u = 2^-24).  A mean over d <= 512 values is at most 16 additions in a lane and 5 between lanes: 21 u of its terms'
magnitude.  So xhat is off by at most 32 u * (|xhat| + r max|x|) (the second term only where a mean is subtracted), a
weight, a rotation's two products and their sum and the reduced angle table's own exactness add less than 8 u of the two
partners: with 64 u * (largest |n| of the row + r max|x| max|w|) every result of a row is covered, plus half a step of the
stored type.  The input gradient r (gh - m1 - xhat m2) has means below max|gh|: 128 u * r max|gh| (1 + max|xhat| + r max|x|) and
half a step.  A weight gradient is a sum over n rows in chains of at most n / (warps) + 64 additions; with n + 64 and the
terms' own 64 u it is off by at most (n + 128) u * sum |g xhat| at worst, and (n / 64 + 256) u is what is asked here: no
kernel has fewer than 64 chains once n is above 64 * 256."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from proteinpredictmachinelearning_b200 import PATH_SIMT, _lib  # noqa: E402
from proteinpredictmachinelearning_b200 import ops  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
gpu = pytest.mark.gpu


def rand(shape, seed, dtype=F32, shift=0.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") + shift).to(dtype)


def strided(x, layout):
    """x [B, L, h, d] in another memory layout: "tokens", "heads" ([B, h, L, d]), "fused" (a column range of wider rows) or "odd" (a
    start and pitches that are odd)."""
    B, L, h, d = x.shape
    if layout == "tokens":
        return x.contiguous()
    if layout == "heads":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "fused":
        buf = torch.full((B, L, (h + 3) * d), -7.0, device="cuda", dtype=x.dtype)
        y = buf[..., 2 * d:(h + 2) * d].unflatten(-1, (h, d))
    else:
        hp = d + 1
        lp = h * hp + 3
        buf = torch.full((B * L * lp + 1,), -7.0, device="cuda", dtype=x.dtype)
        y = torch.as_strided(buf, (B, L, h, d), (L * lp, lp, hp, 1), 1)
    y.copy_(x)
    return y


def turn(x, cos, sin, interleaved, back=False):
    """Rotation in 64 bits; cos, sin [B, L, rot / 2] fp64."""
    half = cos.shape[-1]
    c, s = cos[:, :, None], (-sin if back else sin)[:, :, None]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def table_rows(cos, sin, positions, B, L):
    if cos is None:
        z = torch.zeros((B, L, 0), device="cuda", dtype=torch.float64)
        return z, z
    pos = (torch.arange(L, device="cuda") if positions is None else positions.long()).expand(B, L).clamp(0, cos.shape[0] - 1)
    return cos.double()[pos], sin.double()[pos]


def parts64(x, norm, eps):
    x = x.double()
    mu = x.mean(-1, keepdim=True) if norm == "layer" else 0.0
    r = torch.ones_like(x[..., :1]) if norm == "none" else ((x - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    return (x - mu) * r, r


def half_step(y, dtype):
    info = torch.finfo(dtype)
    return info.eps / 2 * y.abs() + info.smallest_normal * info.eps / 2


def check_forward(got, x, w, norm, eps, cos, sin, interleaved):
    n, r = parts64(x, norm, eps)
    wd = torch.ones(x.shape[-1], device="cuda", dtype=torch.float64) if w is None else w.double()
    want = turn(n * wd, cos, sin, interleaved)
    big = (n * wd).abs().amax(-1, keepdim=True)
    if norm == "layer":
        big = big + r * x.double().abs().amax(-1, keepdim=True) * wd.abs().max()
    over = (got.double() - want).abs() > 64 * U * big + half_step(want, got.dtype)
    assert not over.any(), (int(over.sum()), (got.double() - want).abs().max().item())


def check_backward(dx, dw, x, dy, w, norm, eps, cos, sin, interleaved):
    n, r = parts64(x, norm, eps)
    g = turn(dy.double(), cos, sin, interleaved, back=True)
    gh = g if w is None else g * w.double()
    want = gh
    if norm != "none":
        want = r * (gh - n * (gh * n).mean(-1, keepdim=True) - (gh.mean(-1, keepdim=True) if norm == "layer" else 0.0))
    top = gh.abs().amax(-1, keepdim=True)
    if norm != "none":
        top = r * top * (1 + n.abs().amax(-1, keepdim=True) + (r * x.double().abs().amax(-1, keepdim=True) if norm == "layer" else 0.0))
    over = (dx.double() - want).abs() > 128 * U * top + half_step(want, dx.dtype)
    assert not over.any(), (int(over.sum()), (dx.double() - want).abs().max().item())
    if w is None:
        assert dw is None
        return
    terms = g * n
    scale = terms.abs().sum((0, 1, 2))
    if norm == "layer":
        scale = scale + (g.abs() * r * x.double().abs().amax(-1, keepdim=True)).sum((0, 1, 2))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    off = (dw.double() - terms.sum((0, 1, 2))).abs()
    assert (off <= (rows / 64 + 256) * U * scale).all(), (off / scale).max().item()


@pytest.fixture
def no_device_abort():
    yield
    code, where = ops.device_status()
    assert code == 0, f"a kernel gave up a bounded wait: code {code} at site {where:#x}"


def both(B, L, hq, hk, d, dtype=F32, norm="rms", rot=None, interleaved=False, weights=True, positions=None, rows=None, src="tokens", dst="tokens",
         eps=1e-6, shift=0.0):
    """Forward and backward of one call, checked."""
    rot = d // 2 * 2 if rot is None else rot
    q = strided(rand((B, L, hq, d), 1, dtype, shift), src) if hq else None
    k = strided(rand((B, L, hk, d), 2, dtype, shift), src) if hk else None
    qw, kw = (rand((d,), 3) * 0.3 + 1, rand((d,), 4) * 0.3 + 1) if weights else (None, None)
    cos, sin = ops.rope_table(rows or L, rot) if rot else (None, None)
    how = dict(q_weight=qw if hq else None, k_weight=kw if hk else None, norm=norm, eps=eps, cos=cos, sin=sin, positions=positions,
               interleaved=interleaved)
    out = tuple(None if x is None else strided(torch.full_like(x, 3.0), dst) for x in (q, k))
    qo, ko = ops.qk_norm_rope(q, k, out=out, **how)
    c64, s64 = table_rows(cos, sin, positions, B, L)
    for got, x, w in ((qo, q, how["q_weight"]), (ko, k, how["k_weight"])):
        if x is not None:
            check_forward(got, x, w, norm, eps, c64, s64, interleaved)
    dqo, dko = (strided(rand((B, L, hq, d), 5, dtype), dst) if hq else None, strided(rand((B, L, hk, d), 6, dtype), dst) if hk else None)
    dx = tuple(None if x is None else strided(torch.full_like(x, 3.0), src) for x in (q, k))
    g = ops.qk_norm_rope_backward(q, k, dqo, dko, out=dx, **how)
    for x, dy, w, a, b in ((q, dqo, how["q_weight"], "dQ", "dq_weight"), (k, dko, how["k_weight"], "dK", "dk_weight")):
        if x is not None:
            check_backward(g[a], g.get(b), x, dy, w, norm, eps, c64, s64, interleaved)
    for t in (*out, *dx):                          # what lies between the rows of a strided result stays
        if t is not None and t._base is not None:
            base = t._base.clone()
            torch.as_strided(base, t.shape, t.stride(), t.storage_offset()).fill_(-7.0)
            assert (base == -7).all()
    return g


HEAD_DIMS = [1, 2, 3, 6, 8, 16, 20, 32, 33, 40, 64, 80, 96, 128, 130, 160, 192, 200, 256, 320, 512]


@gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", HEAD_DIMS)
def test_head_dims_and_types(d, dtype, no_device_abort):
    for interleaved in (False, True):
        both(2, 5, 4, 2, d, dtype, interleaved=interleaved)
    both(1, 7, 3, 3, d, dtype, norm="layer", src="fused", dst="heads", shift=0.5)


@gpu
@pytest.mark.parametrize("d,rot", [(64, 0), (64, 2), (64, 16), (64, 24), (64, 62), (80, 32), (80, 20), (128, 96), (128, 4), (40, 6), (33, 10), (256, 128), (8, 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_partial_rotation(d, rot, interleaved, no_device_abort):
    for dtype in (F32, BF16):
        both(2, 9, 4, 1, d, dtype, rot=rot, interleaved=interleaved, src="fused", dst="heads")


@gpu
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("src,dst", [("tokens", "tokens"), ("fused", "heads"), ("heads", "fused"), ("odd", "odd")])
def test_norms_layouts(norm, weights, src, dst, no_device_abort):
    for d, dtype in ((32, F32), (64, BF16), (40, F16)):
        both(3, 17, 6, 2, d, dtype, norm=norm, weights=weights, src=src, dst=dst, shift=0.2)


@gpu
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (32, 8), (7, 1), (1, 0), (0, 5), (64, 1), (3, 16)])
@pytest.mark.parametrize("B,L", [(1, 1), (8, 1), (2, 3), (1, 257), (33, 5)])
def test_head_counts_and_lengths(hq, hk, B, L, no_device_abort):
    for d, dtype in ((128, BF16), (32, F32)):
        both(B, L, hq, hk, d, dtype)


@gpu
@pytest.mark.parametrize("dtype,d,B,L,hq,hk", [(F32, 32, 64, 256, 8, 8), (BF16, 128, 2, 2000, 16, 4), (F16, 80, 3, 777, 12, 3), (BF16, 64, 300, 51, 8, 8)])
def test_many_rows(dtype, d, B, L, hq, hk, no_device_abort):
    both(B, L, hq, hk, d, dtype, src="fused", dst="heads")
    both(B, L, hq, hk, d, dtype, norm="layer", interleaved=True)


@gpu
def test_rows_of_zeros_constants_and_large_values(no_device_abort):
    """Zeros under every norm, a constant row under LayerNorm (variance 0, eps alone), squares near the end of fp32."""
    d = 64
    cos, sin = ops.rope_table(4, d)
    x = torch.zeros((1, 4, 2, d), device="cuda")
    x[0, 1], x[0, 2], x[0, 3] = 5.0, 1e-30, 1e18
    for norm in ("rms", "layer"):
        y, _ = ops.qk_norm_rope(x, None, norm=norm, cos=cos, sin=sin)
        c64, s64 = table_rows(cos, sin, None, 1, 4)
        check_forward(y, x, None, norm, 1e-6, c64, s64, False)
        g = ops.qk_norm_rope_backward(x, None, torch.ones_like(x), None, norm=norm, cos=cos, sin=sin)["dQ"]
        check_backward(g, None, x, torch.ones_like(x), None, norm, 1e-6, c64, s64, False)
    y, _ = ops.qk_norm_rope(torch.zeros((1, 1, 1, d), device="cuda"), None, eps=0.0)
    assert torch.isnan(y).all()                                       # 0 / 0, as the formula says


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinities_and_nan_stay_in_their_row(dtype, no_device_abort):
    q = rand((2, 8, 4, 64), 1, dtype)
    q[0, 1, 2, 5], q[1, 7, 0, 63] = float("nan"), float("inf")
    bad = torch.zeros((2, 8, 4), dtype=torch.bool, device="cuda")
    bad[0, 1, 2] = bad[1, 7, 0] = True
    cos, sin = ops.rope_table(8, 64)
    y, _ = ops.qk_norm_rope(q, None, cos=cos, sin=sin)
    assert torch.isfinite(y[~bad]).all() and torch.isnan(y[0, 1, 2]).all() and torch.isnan(y[1, 7, 0]).any()
    g = ops.qk_norm_rope_backward(q, None, torch.ones_like(q), None, cos=cos, sin=sin)["dQ"]
    assert torch.isfinite(g[~bad]).all() and torch.isnan(g[0, 1, 2]).all()


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 16), (32, 0), (40, 4), (33, 10), (64, 12)])
def test_infinities_and_nan_stay_in_their_pair_without_a_norm(d, rot, interleaved, no_device_abort):
    """Without a norm a value meets its partner of the rotation and nothing else, forward and backward."""
    q = rand((2, 3, 2, d), 1)
    cos, sin = ops.rope_table(3, rot) if rot else (None, None)
    for e, value in ((rot, float("inf")), (d - 1, float("nan")), (rot + 1, float("-inf"))):
        x = q.clone()
        x[0, 2, 1, e] = value
        y, _ = ops.qk_norm_rope(x, None, norm="none", cos=cos, sin=sin, interleaved=interleaved)
        g = ops.qk_norm_rope_backward(q, None, x, None, norm="none", cos=cos, sin=sin, interleaved=interleaved)["dQ"]
        for r in (y, g):
            finite = torch.isfinite(r)
            assert not finite[0, 2, 1, e] and int((~finite).sum()) == 1


@gpu
@pytest.mark.parametrize("d", [64, 40, 33])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_positions_padding_and_the_end_of_the_table(d, dtype, no_device_abort):
    """Positions in any order and twice, shared and per batch; negative ones are padding; one beyond the table gives NaN."""
    B, L, rot, rows = 3, 21, d // 2 * 2, 50
    pos = torch.randint(0, rows, (B, L), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.int32)
    both(B, L, 4, 2, d, dtype, positions=pos, rows=rows)
    both(B, L, 4, 2, d, dtype, positions=pos[0], rows=rows, norm="layer")
    both(B, L, 4, 2, d, dtype, positions=torch.cat((pos, pos), 1)[:, :L], rows=rows)      # rows of a wider tensor
    q, k, w = rand((B, L, 4, d), 1, dtype), rand((B, L, 2, d), 2, dtype), rand((d,), 3) + 1
    cos, sin = ops.rope_table(rows, rot)
    pad = pos.clone()
    pad[0, 4:], pad[2, 0], pad[1, :] = -1, -(1 << 31), -5
    keep = pad >= 0
    how = dict(q_weight=w, k_weight=w, cos=cos, sin=sin)
    out = (torch.full_like(q, 9.0), torch.full_like(k, 9.0))
    ops.qk_norm_rope(q, k, positions=pad, out=out, **how)
    full = ops.qk_norm_rope(q, k, positions=pos, **how)
    for o, f in zip(out, full):
        assert (o[~keep] == 9).all() and torch.equal(o[keep], f[keep])
    dq, dk = rand(q.shape, 5, dtype), rand(k.shape, 6, dtype)
    dq[~keep], dk[~keep] = float("nan"), float("inf")                 # what padding holds does not matter
    q2, k2 = q.clone(), k.clone()
    q2[~keep], k2[~keep] = float("inf"), float("nan")
    g = ops.qk_norm_rope_backward(q2, k2, dq, dk, positions=pad, **how)
    for dx, name, x, dy in ((g["dQ"], "dq_weight", q, dq), (g["dK"], "dk_weight", k, dk)):
        assert not dx[~keep].any()
        c64, s64 = table_rows(cos, sin, pos, B, L)
        c64, s64 = c64[keep][None], s64[keep][None]
        check_backward(dx[keep][None], g[name], x[keep][None], dy[keep][None], w, "rms", 1e-6, c64, s64, False)
    bad = torch.full((d,), float("nan"), device="cuda")
    g = ops.qk_norm_rope_backward(q2, k2, dq, dk, bad, bad, cos=cos, sin=sin, positions=pad)
    assert not g["dQ"][~keep].any() and not g["dK"][~keep].any()      # whatever the weights are
    far = pos.clone()
    far[1, 3], far[2, 20] = rows, 2147483647
    ok = (far >= 0) & (far < rows)
    for o, f in zip(ops.qk_norm_rope(q, k, positions=far, **how), full):
        assert torch.isnan(o[~ok][..., :rot]).all() and torch.equal(o[ok], f[ok])
    g = ops.qk_norm_rope_backward(q, k, rand(q.shape, 5, dtype), rand(k.shape, 6, dtype), positions=far, **how)
    assert torch.isnan(g["dQ"][~ok]).all() and torch.isfinite(g["dQ"][ok]).all() and torch.isnan(g["dq_weight"]).any()


@gpu
def test_in_place_equals_a_new_result(no_device_abort):
    for d, dtype in ((64, BF16), (32, F32), (33, F32), (80, F16)):
        p = rand((2, 19, 10 * d), 1, dtype)
        view = lambda t: (t[..., :6 * d].unflatten(-1, (6, d)), t[..., 6 * d:8 * d].unflatten(-1, (2, d)))     # noqa: E731
        cos, sin = ops.rope_table(19, d // 2 * 2)
        w = rand((d,), 2) + 1
        want = ops.qk_norm_rope(*view(p), q_weight=w, cos=cos, sin=sin)
        mine = p.clone()
        assert torch.equal(ops.qk_norm_rope(*view(mine), q_weight=w, cos=cos, sin=sin, out=(view(p.clone())[0], None))[1], want[1])
        ops.qk_norm_rope(*view(mine), q_weight=w, cos=cos, sin=sin, out=view(mine))
        assert torch.equal(view(mine)[0], want[0]) and torch.equal(view(mine)[1], want[1]) and torch.equal(mine[..., 8 * d:], p[..., 8 * d:])
        dy = rand((2, 19, 10 * d), 3, dtype)
        want = ops.qk_norm_rope_backward(*view(p), *view(dy), q_weight=w, cos=cos, sin=sin)
        got = ops.qk_norm_rope_backward(*view(p), *view(dy), q_weight=w, cos=cos, sin=sin, out=view(dy))
        for n in want:
            assert torch.equal(got[n], want[n])


@gpu
def test_broadcast_inputs(no_device_abort):
    """Inputs and gradients with stride 0; a result with stride 0 is refused."""
    q = rand((1, 6, 1, 64), 1).expand(3, 6, 4, 64)
    cos, sin = ops.rope_table(6, 64)
    y, _ = ops.qk_norm_rope(q, None, cos=cos, sin=sin)
    assert torch.equal(y, ops.qk_norm_rope(q.contiguous(), None, cos=cos, sin=sin)[0])
    w = rand((64,), 2)
    g = ops.qk_norm_rope_backward(q, None, q, None, q_weight=w, cos=cos, sin=sin)
    h = ops.qk_norm_rope_backward(q.contiguous(), None, q.contiguous(), None, q_weight=w, cos=cos, sin=sin)
    assert all(torch.equal(g[n], h[n]) for n in h)
    with pytest.raises(RuntimeError, match="status 1"):
        ops.qk_norm_rope(q.contiguous(), None, cos=cos, sin=sin, out=(q, None))
    with pytest.raises(RuntimeError, match="status 1"):
        ops.qk_norm_rope_backward(q, None, q, None, cos=cos, sin=sin, out=(q, None))


@gpu
@pytest.mark.parametrize("norm,interleaved", [("rms", False), ("layer", True), ("none", False)])
def test_gradients_against_differences(norm, interleaved, no_device_abort):
    """Directional derivatives of sum(dy * f) in 64 bits by central differences (h = 1e-4: truncation h^2 / 6 times the third
    derivative, about 1e-8 of the magnitudes here), for both inputs and both weights."""
    B, L, hq, hk, d, rot = 2, 6, 4, 2, 32, 24
    x, w = [rand((B, L, h, d), i) for i, h in ((1, hq), (2, hk))], [rand((d,), i) * 0.3 + 1 for i in (3, 4)]
    dy, v, vw = [rand(t.shape, 5) for t in x], [rand(t.shape, 7) for t in x], [rand((d,), 8) for _ in w]
    cos, sin = ops.rope_table(L, rot)
    c64, s64 = table_rows(cos, sin, None, B, L)
    g = ops.qk_norm_rope_backward(*x, *dy, q_weight=w[0], k_weight=w[1], norm=norm, eps=1e-5, cos=cos, sin=sin, interleaved=interleaved)
    for i, (a, b) in enumerate((("dQ", "dq_weight"), ("dK", "dk_weight"))):
        def f(t, tw):
            return (turn(parts64(x[i].double() + t * v[i].double(), norm, 1e-5)[0] * (w[i].double() + tw * vw[i].double()), c64, s64, interleaved) *
                    dy[i].double()).sum().item()
        h = 1e-4
        for got, want, size in (((g[a].double() * v[i].double()).sum().item(), (f(h, 0) - f(-h, 0)) / (2 * h), (g[a].abs() * v[i].abs()).sum().item()),
                                ((g[b].double() * vw[i].double()).sum().item(), (f(0, h) - f(0, -h)) / (2 * h), (g[b].abs() * vw[i].abs()).sum().item())):
            assert abs(got - want) <= 1e-5 * size, (a, got, want)


@gpu
def test_offsets_beyond_32_bits(no_device_abort):
    d, h, pitch = 64, 3, (1 << 31) // 3 // 8 * 8
    buf = torch.empty(4 * pitch + h * d, device="cuda", dtype=BF16)
    x = torch.as_strided(buf, (1, 5, h, d), (0, pitch, d, 1))
    x.copy_(rand((1, 5, h, d), 1, BF16))
    cos, sin = ops.rope_table(5, d)
    w = rand((d,), 3) + 1
    want, _ = ops.qk_norm_rope(x.contiguous(), None, q_weight=w, cos=cos, sin=sin)
    back = ops.qk_norm_rope_backward(x.contiguous(), None, x.contiguous(), None, q_weight=w, cos=cos, sin=sin)
    got = ops.qk_norm_rope_backward(x, None, x, None, q_weight=w, cos=cos, sin=sin)
    assert all(torch.equal(got[n], back[n]) for n in back)
    ops.qk_norm_rope(x, None, q_weight=w, cos=cos, sin=sin, out=(x, None))
    assert torch.equal(x, want)


@gpu
def test_last_row_of_a_long_table(no_device_abort):
    """A table row beyond 2^31 elements is looked up there."""
    rows, half = (1 << 31) // 64 + 3, 64
    cos = torch.empty((rows, half), device="cuda")
    sin = torch.empty((rows, half), device="cuda")
    c, s = ops.rope_table(3, 128)
    cos[-3:], sin[-3:] = c, s
    q = rand((1, 3, 2, 128), 1)
    pos = torch.arange(rows - 3, rows, device="cuda", dtype=torch.int32)
    assert torch.equal(ops.qk_norm_rope(q, None, cos=cos, sin=sin, positions=pos)[0], ops.qk_norm_rope(q, None, cos=c, sin=s)[0])


@gpu
def test_empty_batches():
    w = torch.ones(16, device="cuda")
    for shape in ((0, 4, 2, 16), (3, 0, 2, 16)):
        q = torch.empty(shape, device="cuda")
        assert ops.qk_norm_rope(q, q, q_weight=w)[0].shape == shape
        g = ops.qk_norm_rope_backward(q, q, q, q, q_weight=w, k_weight=w)
        assert g["dQ"].shape == shape and not g["dq_weight"].any() and not g["dk_weight"].any()


@gpu
def test_repeated_and_captured_backward_gives_the_same_bits(no_device_abort):
    """Weight gradients do not depend on scheduling; two graphs keep workspaces of their own and replay in turn on another stream."""
    args = [rand((4, 300, h, 64), i, BF16) for i, h in ((1, 8), (2, 2), (3, 8), (4, 2))]
    w = rand((64,), 5) + 1
    cos, sin = ops.rope_table(300, 64)
    how = dict(q_weight=w, k_weight=w, cos=cos, sin=sin)
    want = ops.qk_norm_rope_backward(*args, **how)
    for _ in range(3):
        again = ops.qk_norm_rope_backward(*args, **how)
        assert all(torch.equal(again[n], want[n]) for n in want)
    copies = [[t.clone() for t in args] for _ in range(2)]
    graphs, outs = [], []
    for c in copies:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((ops.qk_norm_rope(c[0], c[1], **how), ops.qk_norm_rope_backward(*c, **how)))
        graphs.append(g)
    for c in copies:
        for t in c:
            t.mul_(-0.5)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for st, g in ((a, graphs[0]), (b, graphs[1]), (b, graphs[1])):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    want = ops.qk_norm_rope_backward(*copies[0], **how)
    y = ops.qk_norm_rope(copies[0][0], copies[0][1], **how)
    for fwd, back in outs:
        assert torch.equal(fwd[0], y[0]) and torch.equal(fwd[1], y[1]) and all(torch.equal(back[n], want[n]) for n in want)


# ---- the operators together --------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("B,L,h,d,c", [(3, 51, 8, 32, 128), (2, 100, 4, 8, 64)])
def test_gated_attention_layer_in_8_bits(B, L, h, d, c, no_device_abort):
    """x -> 8-bit [q | k | v | gate] projection -> norm and rotation in place -> gated attention where the projection lies -> 8-bit
    output projection.  Each stage against 64 bits on the stage before: the attention (exact fp32 path) at the 1e-5 its own
    tests ask, the output projection at its own bound."""
    hd = h * d
    W, ws = ops.quantize_tokens_i8(rand((4 * hd, c), 1) * 0.1)
    Wo, wos = ops.quantize_tokens_i8(rand((c, hd), 2) * 0.05)
    bias, qw, kw = rand((4 * hd,), 3) * 0.1, rand((d,), 4) * 0.2 + 1, rand((d,), 5) * 0.2 + 1
    x = rand((B * L, c), 6, BF16)
    cos, sin = ops.rope_table(L, d)
    p = ops.linear_i8(x, W, ws, bias=bias, dtype=F32).view(B, L, 4 * hd)
    before = p.clone()
    q, k = (p[..., i * hd:(i + 1) * hd].unflatten(-1, (h, d)) for i in (0, 1))
    ops.qk_norm_rope(q, k, qw, kw, cos=cos, sin=sin, out=(q, k))
    o, _ = ops.flash_attn_tokens(p[..., :hd], p[..., hd:2 * hd], p[..., 2 * hd:3 * hd], h, gate=p[..., 3 * hd:], path=PATH_SIMT,
                                 out=torch.empty((B, L, hd), device="cuda"))
    y = ops.linear_i8(o.view(B * L, hd), Wo, wos, dtype=F32)

    c64, s64 = table_rows(cos, sin, None, B, L)
    split = lambda t, i: t[..., i * hd:(i + 1) * hd].unflatten(-1, (h, d))     # noqa: E731
    check_forward(q, split(before, 0), qw, "rms", 1e-6, c64, s64, False)
    check_forward(k, split(before, 1), kw, "rms", 1e-6, c64, s64, False)
    assert torch.equal(p[..., 2 * hd:], before[..., 2 * hd:])
    q64, k64, v64 = (split(p, i).double().transpose(1, 2) for i in (0, 1, 2))
    a64 = torch.softmax(q64 @ k64.transpose(-1, -2) / d ** 0.5, -1) @ v64
    want = a64.transpose(1, 2).reshape(B, L, hd) * torch.sigmoid(p[..., 3 * hd:].double())
    assert ((o.double() - want).abs().max() / want.abs().max()).item() <= 1e-5
    oq, os_ = ops.quantize_tokens_i8(o.view(B * L, hd))
    want = (oq.double() @ Wo.double().t()) * os_.double()[:, None] * wos.double()
    assert ((y.double() - want).abs() <= 16 * U * want.abs() + 1e-30).all()


@gpu
def test_training_step_through_the_attention(no_device_abort):
    """qk_norm_rope into the head-major layout, attention forward and backward (exact fp32), qk_norm_rope_backward; all
    gradients against autograd in 64 bits (1e-4 of the largest, as the attention's own gradients are held to 1e-5 and pass
    through a norm of rows of size about 1)."""
    B, L, h, d = 2, 48, 4, 32
    q, k, v, do = (rand((B, L, h, d), i) for i in (1, 2, 3, 4))
    qw, kw = rand((d,), 5) * 0.2 + 1, rand((d,), 6) * 0.2 + 1
    cos, sin = ops.rope_table(L, d)
    how = dict(q_weight=qw, k_weight=kw, cos=cos, sin=sin)
    heads = lambda t: t.transpose(1, 2).contiguous()     # noqa: E731
    qh, kh = (torch.empty((B, h, L, d), device="cuda") for _ in range(2))
    ops.qk_norm_rope(q, k, out=(qh.transpose(1, 2), kh.transpose(1, 2)), **how)
    o, lse = ops.flash_attn_forward_cuda(qh, kh, heads(v), path=PATH_SIMT)
    a = ops.flash_attn_backward_cuda(qh, kh, heads(v), o, heads(do), lse, want=("dQ", "dK", "dV"))
    g = ops.qk_norm_rope_backward(q, k, a["dQ"].transpose(1, 2), a["dK"].transpose(1, 2), **how)

    c64, s64 = (t[:, :, None] for t in table_rows(cos, sin, None, B, L))
    leaves = [t.double().requires_grad_() for t in (q, k, v, qw, kw)]

    def f(x, w):
        n = x * (x * x).mean(-1, keepdim=True).add(1e-6).rsqrt() * w
        a, b = n[..., :d // 2], n[..., d // 2:]
        return torch.cat((a * c64 - b * s64, b * c64 + a * s64), -1).transpose(1, 2)
    q64, k64 = f(leaves[0], leaves[3]), f(leaves[1], leaves[4])
    o64 = torch.softmax(q64 @ k64.transpose(-1, -2) / d ** 0.5, -1) @ leaves[2].transpose(1, 2)
    want = torch.autograd.grad(o64, leaves, do.double().transpose(1, 2))
    for got, w in zip((g["dQ"], g["dK"], a["dV"].transpose(1, 2), g["dq_weight"], g["dk_weight"]), want):
        assert ((got.double() - w).abs().max() / w.abs().max()).item() <= 1e-4


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_bad_arguments_are_refused_on_the_host(lib):
    p = C.c_void_p(64)
    base = dict(B=2, L=3, hq=4, hk=2, d=16, type=0, norm=1, eps=1e-6, rot=16, interleaved=0, table_rows=3, pos_b=0)
    names = ("Q", "K", "qw", "kw", "cos", "sin", "pos", "Qo", "Ko")

    def view(h, at=64, **kw):
        return C.byref(_lib.Heads(at, kw.get("sb", 3 * h * 16), kw.get("sl", h * 16), kw.get("sh", 16)))
    good = dict(Q=view(4), K=view(2), qw=None, kw=None, cos=p, sin=p, pos=None, Qo=view(4), Ko=view(2))

    def fwd(cfg=None, **kw):
        c = _lib.QkCfg(**{**base, **(cfg or {})})
        return lib.ppml_b200_qk_norm_rope(C.byref(c), *[kw.get(n, good[n]) for n in names], None)

    def bwd(cfg=None, **kw):
        c = _lib.QkCfg(**{**base, **(cfg or {})})
        more = dict(dQ=view(4), dK=view(2), dqw=None, dkw=None, ws=None, bytes=0)
        return lib.ppml_b200_qk_norm_rope_backward(C.byref(c), *[kw.get(n, good[n]) for n in names], *[kw.get(n, v) for n, v in more.items()], None)
    for call in (fwd, bwd):
        for cfg in (dict(B=-1), dict(L=-1), dict(hq=-1), dict(hk=-1), dict(hq=0, hk=0), dict(d=0), dict(type=3), dict(norm=3), dict(norm=-1),
                    dict(rot=-2), dict(rot=3), dict(rot=18), dict(eps=-1.0), dict(eps=float("nan")), dict(table_rows=0), dict(table_rows=2),
                    dict(hq=2147483647, hk=1)):
            assert call(cfg) == 1, cfg
        assert call(dict(d=513, rot=0)) == 9 and call(dict(B=65536, L=32768)) == 9
        for kw in (dict(Q=None), dict(K=None), dict(Qo=None), dict(Ko=None), dict(cos=None), dict(sin=None), dict(Q=view(4, None)), dict(Q=view(4, 66)),
                   dict(K=view(2, sl=-1)), dict(qw=C.c_void_p(65)), dict(cos=C.c_void_p(66)), dict(pos=C.c_void_p(66))):
            assert call(None, **kw) == 1, kw
        assert call(dict(pos_b=-1), pos=p) == 1
        assert call(dict(type=1), Q=view(4, 65)) == 1
    for kw in (dict(Qo=view(4, sh=8)), dict(Qo=view(4, sl=0)), dict(Ko=view(2, sb=0)), dict(Qo=view(4, sb=8))):
        assert fwd(None, **kw) == 1, kw
    for kw in (dict(dQ=None), dict(dK=None), dict(dQ=view(4, sh=8)), dict(dK=view(2, sl=0)), dict(dqw=C.c_void_p(66)), dict(dQ=view(4, 67))):
        assert bwd(None, **kw) == 1, kw
    need = lib.ppml_b200_qk_norm_rope_backward_workspace(C.byref(_lib.QkCfg(**base)))
    assert need > 0 and need % 16 == 0
    for kw in (dict(ws=None, bytes=need), dict(ws=p, bytes=need - 1), dict(ws=C.c_void_p(72), bytes=need)):
        assert bwd(None, dqw=p, **kw) == 3 and bwd(None, dkw=p, **kw) == 3, kw
    assert lib.ppml_b200_qk_norm_rope(None, *[good[n] for n in names], None) == 1
    assert fwd(dict(B=0), Q=None, K=None, Qo=None, Ko=None) == 0 and bwd(dict(L=0), Q=None, K=None, Qo=None, Ko=None, dQ=None, dK=None) == 0


def test_rope_table_in_64_bits():
    cos, sin = ops.rope_table(70000, 64, base=500.0, device="cpu")
    p, i = 69999, np.arange(32)
    want = p * 500.0 ** (-i / 32.0)
    assert cos.shape == (70000, 32) and cos.dtype == F32
    assert np.abs(cos[p].numpy() - np.cos(want)).max() <= U + 70000 * 2.0 ** -52 * 8 and np.abs(sin[p].numpy() - np.sin(want)).max() <= U + 70000 * 2.0 ** -52 * 8
    assert ops.rope_table(3, 0, device="cpu")[0].shape == (3, 0)
    for bad in ((0, 4), (4, 3), (4, -2)):
        with pytest.raises(ValueError):
            ops.rope_table(*bad, device="cpu")


@gpu
def test_wrong_tensors_are_refused():
    q, k, w = rand((2, 5, 4, 16), 1), rand((2, 5, 2, 16), 2), torch.ones(16, device="cuda")
    cos, sin = ops.rope_table(5, 16)
    pos = torch.zeros((2, 5), device="cuda", dtype=torch.int32)
    for bad in (lambda: ops.qk_norm_rope(None, None), lambda: ops.qk_norm_rope(q.cpu(), None), lambda: ops.qk_norm_rope(q[0], None),
                lambda: ops.qk_norm_rope(q.double(), None), lambda: ops.qk_norm_rope(q, k[:1]), lambda: ops.qk_norm_rope(q, k[..., :8]),
                lambda: ops.qk_norm_rope(q, k.half()), lambda: ops.qk_norm_rope(q.transpose(2, 3), None), lambda: ops.qk_norm_rope(q, k, norm="l2"),
                lambda: ops.qk_norm_rope(q, k, q_weight=w[:8]), lambda: ops.qk_norm_rope(q, k, q_weight=w.half()), lambda: ops.qk_norm_rope(q, k, cos=cos),
                lambda: ops.qk_norm_rope(q, k, cos=cos, sin=sin[:, :4]), lambda: ops.qk_norm_rope(q, k, cos=cos.double(), sin=sin.double()),
                lambda: ops.qk_norm_rope(q, k, cos=cos, sin=sin, positions=pos.long()), lambda: ops.qk_norm_rope(q, k, cos=cos, sin=sin, positions=pos[:, :4]),
                lambda: ops.qk_norm_rope(q, k, cos=cos.cpu(), sin=sin.cpu()), lambda: ops.qk_norm_rope(q, k, eps="1"), lambda: ops.qk_norm_rope(q, k, interleaved=q),
                lambda: ops.qk_norm_rope(q, [k]),
                lambda: ops.qk_norm_rope(q, None, out=(q, k)), lambda: ops.qk_norm_rope(q, k, out=(q, q)), lambda: ops.qk_norm_rope(q, k, out=(q.half(), k)),
                lambda: ops.qk_norm_rope_backward(q, k, q, None), lambda: ops.qk_norm_rope_backward(q, k, q, k[:, :3])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="status 1"):
        ops.qk_norm_rope(q, k, cos=cos[:4], sin=sin[:4])              # five tokens, four rows, no positions
    with pytest.raises(RuntimeError, match="status 9"):
        ops.qk_norm_rope(rand((1, 1, 1, 514), 1), None)
