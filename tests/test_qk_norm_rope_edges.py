"""Norms of queries and keys with the position rotation at the edges: table rows that no token looks up."""
import pytest

torch = pytest.importorskip("torch")

from proteinpredictmachinelearning_b200 import ops  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def rand(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


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
