"""Norms of queries and keys with the position rotation at the edges: table rows that no token looks up; every instance
against 64 bits with checks that a NaN fails."""
import pytest

torch = pytest.importorskip("torch")

from proteinpredictmachinelearning_b200 import ops  # noqa: E402
from test_qk_norm_rope import half_step, parts64, table_rows, turn  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def rand(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


U = 2.0 ** -24


def check(got, want, tol):
    """NaN fails, in what is wanted too."""
    assert torch.isfinite(want).all()
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (int((~(off <= tol)).sum()), off.max().item())


# chunks of 16 bytes with 1 to 32 lanes a row, of 8 and of 4 bytes, and the element-wise kernel (33)
@gpu
@pytest.mark.parametrize("dtype,d", [(F32, 8), (F32, 16), (F32, 32), (F32, 64), (F32, 128), (F32, 256), (F32, 12), (F32, 6), (F32, 33),
                                     (BF16, 16), (BF16, 32), (BF16, 64), (BF16, 128), (BF16, 256), (BF16, 512), (BF16, 40), (BF16, 20), (BF16, 33),
                                     (F16, 64), (F16, 80), (F16, 36)])
@pytest.mark.parametrize("norm,interleaved", [("rms", False), ("layer", True), ("none", False)])
def test_rows_of_the_table_that_no_token_looks_up(dtype, d, norm, interleaved):
    """A first row that is not finite changes nothing while live positions begin at 1, with idle lanes behind the last token, with
    padding among the tokens, and with nothing but padding."""
    rot, rows = d // 2 * 2, 50
    w = rand((d,), 3) + 1
    cos, sin = ops.rope_table(rows, rot)
    for B, L, hq, hk in ((1, 1, 1, 1), (1, 5, 4, 2), (3, 13, 3, 8)):
        q, k, dq, dk = (rand((B, L, h, d), i, dtype) for i, h in ((1, hq), (2, hk), (5, hq), (6, hk)))
        pos = 1 + torch.arange(B * L, device="cuda", dtype=torch.int32).view(B, L)
        some, none = pos.clone(), torch.full_like(pos, -1)
        some[:, ::3] = -7
        for positions in (pos, some, none):
            how = dict(q_weight=w, k_weight=w, norm=norm, sin=sin, positions=positions, interleaved=interleaved)
            out = (torch.full_like(q, 9.0), torch.full_like(k, 9.0))
            y = ops.qk_norm_rope(q, k, cos=cos, out=tuple(t.clone() for t in out), **how)
            g = ops.qk_norm_rope_backward(q, k, dq, dk, cos=cos, **how)
            assert all(torch.isfinite(t).all() for t in (*y, *g.values()))
            for bad in (float("nan"), float("inf")):
                cos_bad, sin_bad = cos.clone(), sin.clone()
                cos_bad[0], sin_bad[0] = bad, bad
                how["sin"] = sin_bad
                for a, b in zip(y, ops.qk_norm_rope(q, k, cos=cos_bad, out=tuple(t.clone() for t in out), **how)):
                    assert torch.equal(a, b)
                h = ops.qk_norm_rope_backward(q, k, dq, dk, cos=cos_bad, **how)
                for n in g:
                    assert torch.equal(g[n], h[n]), n


@gpu
@pytest.mark.parametrize("dtype,d", [(F32, 8), (F32, 16), (F32, 32), (F32, 64), (F32, 128), (F32, 256), (F32, 512), (F32, 12), (F32, 6), (F32, 33), (F32, 80),
                                     (BF16, 16), (BF16, 32), (BF16, 64), (BF16, 128), (BF16, 256), (BF16, 512), (BF16, 40), (BF16, 20), (BF16, 33), (BF16, 46),
                                     (F16, 64), (F16, 80), (F16, 36), (F16, 96)])
@pytest.mark.parametrize("norm,interleaved,part", [("rms", False, 1), ("layer", True, 1), ("none", False, 1), ("rms", True, 2), ("layer", False, 4)])
def test_every_instance_gives_finite_results(dtype, d, norm, interleaved, part):
    """Results, input gradients and weight gradients of every width of access and number of lanes.  A mean over d <= 512 values is at most
    21 additions deep, with the reciprocal root, the weight and the rotation below 64 u of the row's largest value (under LayerNorm of
    the largest input too); an input gradient below 128 u of r max|g w| (1 + max|xhat|) with the same addition; a weight gradient of n
    rows is no sum of more than n additions, 64 u a term."""
    rot, B, L, hq, hk = d // part // 2 * 2, 2, 19, 5, 2
    cos, sin = ops.rope_table(L, rot) if rot else (None, None)
    c64, s64 = table_rows(cos, sin, None, B, L)
    w = [rand((d,), 3) * 0.3 + 1, rand((d,), 4) * 0.3 + 1]
    x, dy = ([rand((B, L, h, d), i + j, dtype) for j, h in ((0, hq), (1, hk))] for i in (1, 5))
    how = dict(q_weight=w[0], k_weight=w[1], norm=norm, cos=cos, sin=sin, interleaved=interleaved)
    y, g = ops.qk_norm_rope(*x, **how), ops.qk_norm_rope_backward(*x, *dy, **how)
    for i, (dx, dw) in enumerate((("dQ", "dq_weight"), ("dK", "dk_weight"))):
        n, r = parts64(x[i], norm, 1e-6)
        wd, raw = w[i].double(), r * x[i].double().abs().amax(-1, keepdim=True) if norm == "layer" else 0.0
        want = turn(n * wd, c64, s64, interleaved)
        check(y[i], want, 64 * U * ((n * wd).abs().amax(-1, keepdim=True) + raw * wd.abs().max()) + half_step(want, dtype))
        gr = turn(dy[i].double(), c64, s64, interleaved, back=True)
        gh = gr * wd
        want, top = gh, gh.abs().amax(-1, keepdim=True)
        if norm != "none":
            want = r * (gh - n * (gh * n).mean(-1, keepdim=True) - (gh.mean(-1, keepdim=True) if norm == "layer" else 0.0))
            top = r * top * (1 + n.abs().amax(-1, keepdim=True) + raw)
        check(g[dx], want, 128 * U * top + half_step(want, dtype))
        terms = gr * n
        check(g[dw], terms.sum((0, 1, 2)), (B * L * x[i].shape[2] + 64) * U * (terms.abs() + gr.abs() * raw).sum((0, 1, 2)))
