"""What a program asks of the operators around the token-major attention, as timed cases: Linears in 8-bit integers with a
scale for each token and each output channel, and the norms of queries and keys for each head with the position rotation in
the same pass, forward and backward.

`run` computes a case in plain torch operations, or, where `own` is true, through the framework's entry points.  Sizes are
those of the model's blocks (256 residues, MSA depth 256: 65536 tokens, 8 heads of 32; development size 51 residues x 8 rows:
408 tokens) and generic ones for serving (one token, some tens of tokens) and for long sequences.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one token of a serving program through one Linear: the smallest call, latency and launches
        dict(name="i8_linear_one_token", kind="linear", type="bf16", tokens=1, k=1024, n=4096, bias=True, act="none", gate=False),
        # some tens of sequences served together: the weights are the traffic
        dict(name="i8_linear_served_batch", kind="linear", type="bf16", tokens=48, k=4096, n=8192, bias=False, act="none", gate=False),
        # feed-forward up projection over a long batch: the products are the work
        dict(name="i8_linear_wide", kind="linear", type="bf16", tokens=16384, k=4096, n=8192, bias=True, act="gelu", gate=False),
        # gated feed-forward with sizes that end inside every tile
        dict(name="i8_linear_ragged_gated", kind="linear", type="fp16", tokens=1999, k=1000, n=777, bias=True, act="silu", gate=True),
        # query, key-value and gate projections of an MSA attention from one quantized input, development size
        dict(name="i8_projections_dev", kind="projections", type="fp32", tokens=408, k=128, n=128),
        # the same over all 65536 tokens of the full-size MSA
        dict(name="i8_projections_msa", kind="projections", type="fp32", tokens=65536, k=256, n=256),
        # one new token each of eight sequences, far positions, shared key heads
        dict(name="qk_one_token", kind="qk", type="bf16", batch=8, l=1, hq=32, hk=8, d=128, rot=128, norm="rms", pairs="halves",
             source="fused", out="tokens", positions="far"),
        # MSA row attention: queries and keys as they lie in the fused projection
        dict(name="qk_msa_rows", kind="qk", type="fp32", batch=256, l=256, hq=8, hk=8, d=32, rot=32, norm="rms", pairs="halves",
             source="fused", out="tokens", positions="order"),
        # long sequences, result in the head-major layout of the 16-bit attention
        dict(name="qk_long", kind="qk", type="bf16", batch=2, l=16384, hq=32, hk=8, d=128, rot=128, norm="rms", pairs="halves",
             source="fused", out="heads", positions="order"),
        # training step on MSA rows: outputs, input gradients, weight gradients, exact fp32
        dict(name="qk_train_msa_rows", kind="qk_train", type="fp32", batch=64, l=256, hq=8, hk=8, d=32, rot=32, norm="rms",
             pairs="halves", source="dense", out="heads", positions="order"),
        # training step on long sequences, LayerNorm heads, neighbouring pairs
        dict(name="qk_train_long", kind="qk_train", type="bf16", batch=4, l=4096, hq=16, hk=16, d=64, rot=64, norm="layer",
             pairs="neighbours", source="fused", out="tokens", positions="chains"),
        # training step with a head dim that is no power of two, part of it rotated, odd lengths, shared key heads
        dict(name="qk_train_ragged", kind="qk_train", type="fp16", batch=3, l=777, hq=12, hk=3, d=80, rot=32, norm="rms",
             pairs="halves", source="dense", out="tokens", positions="chains"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "projections", "qk", "qk", "qk_train", "qk_train"])
    if kind == "linear":
        k, n = (rng.choice([_log(rng, 40, 8192), 16 * _log(rng, 4, 512), 256, 1024]) for _ in range(2))
        top = min(16384, (1 << 39) // (k * n), (1 << 26) // max(k, n))
        tokens = rng.choice([_log(rng, 1, 16), _log(rng, 8, min(512, top)), _log(rng, 1, top), _log(rng, max(1, top // 16), top)])
        return dict(kind=kind, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), tokens=tokens, k=k, n=n, bias=rng.random() < 0.6,
                    act=rng.choice(["none", "none", "sigmoid", "silu", "gelu", "tanh", "relu"]), gate=rng.random() < 0.3)
    if kind == "projections":
        return dict(kind=kind, type=rng.choice(["fp32", "fp32", "bf16"]), tokens=_log(rng, 60, 65536),
                    k=rng.choice([64, 128, 256, 4 * _log(rng, 8, 64), _log(rng, 30, 256)]),
                    n=rng.choice([64, 128, 256, 8 * _log(rng, 4, 32), _log(rng, 20, 256)]))
    d = rng.choice([32, 32, 64, 64, 128, 128, 8, 16, 40, 80, 96, 256, 2 * _log(rng, 4, 100)])
    rot = d if rng.random() < 0.7 else 2 * rng.randint(0, d // 2)
    hk = rng.choice([1, 2, 4, 8, 8, _log(rng, 1, 16)])
    hq = hk * rng.choice([1, 1, 2, 4])
    top = (1 << (26 if kind == "qk" else 25)) // ((hq + hk) * d)
    tokens = _log(rng, 1, top) if rng.random() < 0.6 else _log(rng, max(1, top // 16), top)
    l = rng.choice([1, _log(rng, 1, 16384), _log(rng, 1, 16384), 256, 51])
    l = min(l, tokens)
    return dict(kind=kind, type=rng.choice(["fp32", "bf16", "bf16", "fp16"]), batch=max(1, tokens // l), l=l, hq=hq, hk=hk, d=d, rot=rot,
                norm=rng.choice(["rms", "rms", "layer", "none"]), pairs=rng.choice(["halves", "halves", "neighbours"]),
                source=rng.choice(["fused", "dense"]), out=rng.choice(["tokens", "heads"]), positions=rng.choice(["order", "chains", "far"]))


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _inputs(c, seed):
    """The tensors of a case: activations behind a LayerNorm (unit variance, some columns larger, as trained models have
    them), Linear weights N(0, 0.02), norm weights around 1, upstream gradients of unit variance."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ty = TYPES[c["type"]]

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale)

    if c["kind"] in ("linear", "projections"):
        T, K, N = c["tokens"], c["k"], c["n"]
        wide = torch.exp(randn(K, scale=0.5))
        t = dict(x=(randn(T, K) * wide).to(ty))
        if c["kind"] == "linear":
            t["w"] = randn(N, K, scale=0.02)
            t["bias"] = randn(N, scale=0.1) if c["bias"] else None
            t["gate"] = randn(T, N).to(ty) if c["gate"] else None
        else:                                      # query; key and value; gate
            t["w"] = [randn(n, K, scale=0.02) for n in (N, 2 * N, N)]
            t["bias"] = randn(N, scale=0.1)
        return t
    B, L, hq, hk, d, rot = (c[n] for n in ("batch", "l", "hq", "hk", "d", "rot"))
    if c["source"] == "fused":                     # column ranges of one projection's output [q | k | v]
        p = randn(B, L, (hq + 2 * hk) * d).to(ty)
        q, k = p[..., :hq * d].unflatten(-1, (hq, d)), p[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    else:
        q, k = randn(B, L, hq, d).to(ty), randn(B, L, hk, d).to(ty)
    t = dict(q=q, k=k, qw=randn(d, scale=0.2).add_(1.0) if c["norm"] != "none" else None,
             kw=randn(d, scale=0.2).add_(1.0) if c["norm"] != "none" else None)
    rows, first = L, torch.arange(L, device="cuda")
    t["pos"] = None
    if c["positions"] == "far":                    # sequences that have run for a while
        rows = max(65536, L)
        t["pos"] = first[None] + torch.randint(0, rows - L + 1, (B, 1), generator=g, device="cuda")
    elif c["positions"] == "chains":               # two chains in a row of residues, the second numbered on behind a gap
        rows = L + 200
        t["pos"] = first[None] + 200 * (first[None] >= torch.randint(0, L + 1, (B, 1), generator=g, device="cuda"))
    if t["pos"] is not None:
        t["pos"] = t["pos"].to(torch.int32)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1))
    t["cos"], t["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    if c["kind"] == "qk_train":
        shape = (lambda h: (B, L, h, d)) if c["out"] == "tokens" else (lambda h: (B, h, L, d))
        t["dq"], t["dk"] = randn(*shape(hq)).to(ty), randn(*shape(hk)).to(ty)
    return t


def _quantize_weights(w):
    """Once per layer: int8 rows, padded in memory to 16 bytes, and the scale of each row."""
    n, k = w.shape
    scale = w.abs().amax(1) / 127.0
    q = torch.zeros((n, (k + 15) // 16 * 16), device=w.device, dtype=torch.int8)[:, :k]
    q.copy_(torch.round(w / scale[:, None]).clamp_(-127, 127))
    return q, scale


def prepare(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "linear":
        t["w"] = _quantize_weights(t["w"])
    elif case["kind"] == "projections":
        t["w"] = [_quantize_weights(w) for w in t["w"]]
    return dict(case), t


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _plain_quantize(x):
    """The largest magnitude of a token becomes 127: integers (as fp32 values) and scales."""
    x = x.float()
    amax = x.abs().amax(1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    return torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-127, 127), scale


def _plain_act(x, act):
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    if act == "tanh":
        return torch.tanh(x)
    return x.clamp(min=0) if act == "relu" else x


def _plain_product(q, scale, w, bias, gate, act, ty):
    y = (q @ w[0].float().t()) * scale * w[1]
    if bias is not None:
        y = y + bias
    y = _plain_act(y, act)
    return (y if gate is None else y * gate.float()).to(ty)


def _rotate(x, cos, sin, pairs, sign):
    """x [B, L, h, d]; cos, sin [.., L, rot / 2]; sign -1 turns back."""
    half = cos.shape[-1]
    cos, sin = cos[..., None, :], sign * sin[..., None, :]
    if pairs == "halves":
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)
    a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., 2 * half:]), -1)


def _normed(x, norm):
    if norm == "none":
        return x, torch.ones_like(x[..., :1])
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _plain_qk(x, w, cos, sin, c):
    n = _normed(x.float(), c["norm"])[0]
    return _rotate(n if w is None else n * w, cos, sin, c["pairs"], 1).to(x.dtype)


def _plain_qk_backward(x, dy, w, cos, sin, c):
    n, r = _normed(x.float(), c["norm"])
    g = _rotate(dy.float(), cos, sin, c["pairs"], -1)
    if c["norm"] == "none":
        return g.to(x.dtype), None
    dw = (g * n).sum((0, 1, 2))
    g = g * w
    dx = g - n * (g * n).mean(-1, keepdim=True)
    if c["norm"] == "layer":
        dx = dx - g.mean(-1, keepdim=True)
    return (dx * r).to(x.dtype), dw


def _plain(c, t):
    if c["kind"] == "linear":
        return _plain_product(*_plain_quantize(t["x"]), t["w"], t["bias"], t["gate"], c["act"], TYPES[c["type"]])
    if c["kind"] == "projections":
        q, s = _plain_quantize(t["x"])
        ty = TYPES[c["type"]]
        return (_plain_product(q, s, t["w"][0], None, None, "none", ty), _plain_product(q, s, t["w"][1], None, None, "none", ty),
                _plain_product(q, s, t["w"][2], t["bias"], None, "sigmoid", ty))
    pos = t["pos"].long() if t["pos"] is not None else torch.arange(c["l"], device="cuda")
    cos, sin = t["cos"][pos], t["sin"][pos]
    q, k = _plain_qk(t["q"], t["qw"], cos, sin, c), _plain_qk(t["k"], t["kw"], cos, sin, c)
    if c["out"] == "heads":
        q, k = q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous()
    if c["kind"] == "qk":
        return q, k
    dq, dk = (t["dq"], t["dk"]) if c["out"] == "tokens" else (t["dq"].transpose(1, 2), t["dk"].transpose(1, 2))
    dq, dqw = _plain_qk_backward(t["q"], dq, t["qw"], cos, sin, c)
    dk, dkw = _plain_qk_backward(t["k"], dk, t["kw"], cos, sin, c)
    return (q, k, dq, dk) if dqw is None else (q, k, dq, dk, dqw, dkw)


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _own(c, t):
    from proteinpredictmachinelearning_b200 import ops
    if c["kind"] == "linear":
        return ops.linear_i8(t["x"], t["w"][0], t["w"][1], bias=t["bias"], gate=t["gate"], act=c["act"])
    if c["kind"] == "projections":
        q, s = ops.quantize_tokens_i8(t["x"])
        ty = TYPES[c["type"]]
        return (ops.mul_mat_i8(q, s, *t["w"][0], dtype=ty), ops.mul_mat_i8(q, s, *t["w"][1], dtype=ty),
                ops.mul_mat_i8(q, s, *t["w"][2], bias=t["bias"], act="sigmoid", dtype=ty))
    B, L, hq, hk, d = (c[n] for n in ("batch", "l", "hq", "hk", "d"))
    how = dict(q_weight=t["qw"], k_weight=t["kw"], norm=c["norm"], eps=EPS, cos=t["cos"], sin=t["sin"], positions=t["pos"],
               interleaved=c["pairs"] == "neighbours")
    if c["out"] == "tokens":
        q, k = ops.qk_norm_rope(t["q"], t["k"], **how)
    else:
        q, k = (torch.empty((B, h, L, d), device="cuda", dtype=TYPES[c["type"]]) for h in (hq, hk))
        ops.qk_norm_rope(t["q"], t["k"], out=(q.transpose(1, 2), k.transpose(1, 2)), **how)
    if c["kind"] == "qk":
        return q, k
    dq, dk = (t["dq"], t["dk"]) if c["out"] == "tokens" else (t["dq"].transpose(1, 2), t["dk"].transpose(1, 2))
    g = ops.qk_norm_rope_backward(t["q"], t["k"], dq, dk, **how)
    return (q, k, g["dQ"], g["dK"]) if t["qw"] is None else (q, k, g["dQ"], g["dK"], g["dq_weight"], g["dk_weight"])


def run(state):
    c, t = state
    return _own(c, t) if own else _plain(c, t)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    c = case
    e = 4 if c["type"] == "fp32" else 2
    if c["kind"] in ("linear", "projections"):
        T, K, N = c["tokens"], c["k"], c["n"]
        if c["kind"] == "projections":
            return dict(bytes=e * T * K + 4 * N * (K + 4) + 4 * N + e * T * 4 * N, flops=2 * T * K * 4 * N)
        return dict(bytes=e * T * K + N * (K + 4) + (4 * N if c["bias"] else 0) + e * T * N * (2 if c["gate"] else 1), flops=2 * T * K * N)
    T, h, d, rot = c["batch"] * c["l"], c["hq"] + c["hk"], c["d"], c["rot"]
    rows = T if c["positions"] == "far" else min(T, c["l"] + (200 if c["positions"] == "chains" else 0))
    table = 4 * rows * rot + (0 if c["positions"] == "order" else 4 * T) + (0 if c["norm"] == "none" else 8 * d)
    if c["kind"] == "qk":
        return dict(bytes=2 * e * T * h * d + table, flops=T * h * (5 * d + 3 * rot))
    return dict(bytes=4 * e * T * h * d + table + (0 if c["norm"] == "none" else 8 * d), flops=T * h * (17 * d + 6 * rot))


# ---- 64-bit results ----------------------------------------------------------------------------------------------------
def _exact_act(y, act):
    return {"none": lambda v: v, "sigmoid": torch.special.expit, "silu": lambda v: v * torch.special.expit(v), "tanh": torch.tanh,
            "relu": lambda v: torch.maximum(v, torch.zeros_like(v)),
            "gelu": lambda v: v * torch.special.expit(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}[act](y)


def _exact_qk(x, w, angle, c):
    """The rotation as a product of complex numbers, from the fp32 table; gradients of this by autograd."""
    d, rot = c["d"], c["rot"]
    if c["norm"] == "layer":
        x = x - x.sum(-1, keepdim=True) / d
    if c["norm"] != "none":
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / d + EPS) * w
    axis = -2 if c["pairs"] == "halves" else -1
    pairs = x[..., :rot].unflatten(-1, (2, rot // 2) if c["pairs"] == "halves" else (rot // 2, 2))
    z = torch.complex(pairs.select(axis, 0), pairs.select(axis, 1)) * angle[..., None, :]
    turn = torch.stack((z.real, z.imag), axis)
    return torch.cat((turn.flatten(-2), x[..., rot:]), -1)


def exact(case, seed):
    c, t = prepare(case, seed)
    if c["kind"] in ("linear", "projections"):
        # the integers and scales are the format's own, defined in fp32; everything behind them in 64 bits
        x = t["x"].float()
        top = x.abs().max(dim=1).values
        s = torch.div(top, torch.tensor(127.0, device="cuda").expand_as(top))
        q = torch.div(x, s[:, None]).nan_to_num(0.0).round().clamp(-127, 127).double()
        step = max(1, (1 << 28) // max(c["k"], 4 * c["n"]))

        def product(w, bias, gate, act):
            wd = w[0].double() * w[1].double()[:, None]
            parts = []
            for i in range(0, c["tokens"], step):
                y = (q[i:i + step] @ wd.t()) * s[i:i + step, None].double()
                y = _exact_act(y if bias is None else y + bias.double(), act)
                parts.append(y if gate is None else y * gate[i:i + step].double())
            return torch.cat(parts)

        if c["kind"] == "linear":
            return product(t["w"], t["bias"], t["gate"], c["act"])
        return product(t["w"][0], None, None, "none"), product(t["w"][1], None, None, "none"), product(t["w"][2], t["bias"], None, "sigmoid")
    pos = torch.arange(c["l"], device="cuda").expand(c["batch"], -1) if t["pos"] is None else t["pos"].long()
    angle = torch.complex(t["cos"].double(), t["sin"].double())[pos]
    out, grads, sums = [], [], []
    for x, w, dy in ((t["q"], t["qw"], t.get("dq")), (t["k"], t["kw"], t.get("dk"))):
        x = x.double().requires_grad_(dy is not None)
        w = None if w is None else w.double().requires_grad_(dy is not None)
        y = _exact_qk(x, w, angle, c)
        y = y if c["out"] == "tokens" else y.transpose(1, 2)
        out.append(y.detach().contiguous())
        if dy is not None:
            g = torch.autograd.grad(y, [x] if w is None else [x, w], dy.double())
            grads.append(g[0])
            sums += [] if w is None else [g[1]]
    return tuple(out + grads + sums)
