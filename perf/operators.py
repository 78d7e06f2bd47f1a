"""The measured cases of the token operators: fused linear layers, query / key normalisation with the position
rotation, and attention over packed documents, each forwards and backwards.

Tokens of several frames (or streams) are packed one after another; a frame is a document, and cumulative offsets say
where each begins.  ``run`` with ``own`` false computes the operators in elementary torch operations in 32 bits, with
one rounding at the end; with ``own`` true it calls ``promptmoge_b200.tokens``.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: multiply-adds of the largest listed product; drawn cases stay below
MOST_MACS = 38400 * 1024 * 4096
#: score entries times the head size of the largest listed attention, padding included; drawn cases stay below
MOST_SCORES = 16 * 16 * 1200 * 1200 * 64


def listed():
    return [
        # one token of a stream through the block's expanding layer: what a token-by-token caller waits for
        dict(name="linear_token", op="linear", grad=False, rows=1, k=1024, n=4096, dtype="bf16", act="gelu",
             bias=True, residual=False, save=False),
        # one frame's 30x40 encoder tokens with their two UV channels: rows of 1026 values, not a multiple of 16 bytes
        dict(name="linear_uv", op="linear", grad=False, rows=1200, k=1026, n=1024, dtype="fp16", act="silu",
             bias=True, residual=True, save=False),
        # a batch of 32 frames through the expanding layer
        dict(name="linear_frames", op="linear", grad=False, rows=38400, k=1024, n=4096, dtype="bf16", act="gelu",
             bias=True, residual=False, save=False),
        # the same layer's gradients for 8 frames: input, weight, bias
        dict(name="linear_grad", op="linear", grad=True, rows=9600, k=1024, n=4096, dtype="bf16", act="gelu",
             bias=True, residual=False, save=False),
        # sixteen streams, one new token each
        dict(name="rope_token", op="rope", grad=False, rows=16, hq=16, hk=4, d=64, rot=64, dtype="bf16",
             interleaved=False, weight=True),
        # queries and keys of 32 frames, read in place from the fused projection
        dict(name="rope_frames", op="rope", grad=False, rows=38400, hq=16, hk=4, d=64, rot=64, dtype="bf16",
             interleaved=False, weight=True),
        # their gradients at a head of 128 with interleaved pairs and an odd number of tokens
        dict(name="rope_grad", op="rope", grad=True, rows=19201, hq=16, hk=4, d=128, rot=96, dtype="fp16",
             interleaved=True, weight=True),
        # 32 streams, one new token each, over caches of up to 8192 tokens
        dict(name="attn_token", op="attention", grad=False, docs=32, max_q=1, max_k=8192, ragged=True, cache=True,
             hq=16, hk=4, d=64, dtype="bf16", causal=True, prefix=0, softcap=0.0, bias=False, lens=1),
        # one stream alone, four drafted tokens over a long cache with the distance bias
        dict(name="attn_long", op="attention", grad=False, docs=1, max_q=4, max_k=65501, ragged=False, cache=True,
             hq=16, hk=4, d=128, dtype="fp16", causal=True, prefix=0, softcap=0.0, bias=True, lens=2),
        # 16 frames of up to 30x40 tokens, each attending within itself
        dict(name="attn_frames", op="attention", grad=False, docs=16, max_q=1200, max_k=1200, ragged=True,
             cache=False, hq=16, hk=16, d=64, dtype="fp16", causal=False, prefix=0, softcap=0.0, bias=False, lens=3),
        # two long documents: 1200 prompt tokens seen by all, the rest causal, scores capped
        dict(name="attn_prefix", op="attention", grad=False, docs=2, max_q=2560, max_k=2560, ragged=False,
             cache=False, hq=16, hk=4, d=128, dtype="bf16", causal=True, prefix=1200, softcap=30.0, bias=False,
             lens=4),
        # gradients over 8 frames with the distance bias and shared key heads
        dict(name="attn_grad", op="attention", grad=True, docs=8, max_q=1200, max_k=1200, ragged=True, cache=False,
             hq=16, hk=4, d=64, dtype="bf16", causal=False, prefix=0, softcap=0.0, bias=True, lens=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "rope", "attention", "attention"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "linear":
        grad = rng.random() < 0.4
        k, n = _log(rng, 16, 4096), _log(rng, 16, 4096)
        if rng.random() < 0.6:            # widths are mostly round
            k = max(64, k // 64 * 64)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        rows = min(_log(rng, 1, 38400), max(1, MOST_MACS // (3 if grad else 1) // (k * n)))
        return dict(op=op, grad=grad, rows=rows, k=k, n=n, dtype=dtype,
                    act=rng.choice(["none", "relu", "silu", "gelu"]), bias=rng.random() < 0.8,
                    residual=not grad and rng.random() < 0.5, save=not grad and rng.random() < 0.3)
    if op == "rope":
        d = rng.choice([32, 64, 80, 128])
        hk = rng.choice([1, 2, 4, 8])
        return dict(op=op, grad=rng.random() < 0.5, rows=_log(rng, 1, 19200), hq=hk * rng.choice([1, 2, 4]), hk=hk,
                    d=d, rot=rng.choice([d, d // 2]), dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    interleaved=rng.random() < 0.5, weight=rng.random() < 0.8)
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 4])
    d = rng.choice([32, 64, 80, 128])
    mode = rng.choice(["token", "tile", "grad"])
    softcap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if mode == "token":
        docs, max_q, max_k = _log(rng, 1, 64), rng.choice([1, 1, 2, 5]), _log(rng, 1, 32768)
        max_k = max(max_q, min(max_k, MOST_SCORES // 4 // (docs * hq * d * max_q), 1 << 20))
        while docs * max_k > 1 << 19:
            max_k = max(max_q, max_k // 2)
        return dict(op=op, grad=False, docs=docs, max_q=max_q, max_k=max_k, ragged=rng.random() < 0.7, cache=True,
                    hq=hq, hk=hk, d=d, dtype=dtype, causal=rng.random() < 0.7, prefix=0, softcap=softcap,
                    bias=rng.random() < 0.3, lens=rng.randrange(1 << 20))
    docs = _log(rng, 1, 200)
    max_q = _log(rng, 1, 4096)
    most = MOST_SCORES // (3 if mode == "grad" else 1)
    max_q = max(1, min(max_q, math.isqrt(most // (docs * hq * d))))
    causal = rng.random() < 0.6
    return dict(op=op, grad=mode == "grad", docs=docs, max_q=max_q, max_k=max_q, ragged=rng.random() < 0.7,
                cache=False, hq=hq, hk=hk, d=d, dtype=dtype, causal=causal,
                prefix=rng.randrange(1, max_q + 1) if causal and rng.random() < 0.4 else 0, softcap=softcap,
                bias=rng.random() < 0.4, lens=rng.randrange(1 << 20))


def _lengths(case):
    """Documents' query and key lengths, and their prefixes: a case's own, the same for every seed."""
    r = random.Random(case["lens"])
    docs, mq, mk = case["docs"], case["max_q"], case["max_k"]
    if case["cache"]:
        lq = [mq] * docs
        lk = [r.randint(max(mq, mk // 4), mk) if case["ragged"] else mk for _ in range(docs)]
    else:
        lq = [r.randint(max(0, mq // 3), mq) if case["ragged"] else mq for _ in range(docs)]
        lq[0] = mq
        lk = list(lq)
    return lq, lk, [min(case["prefix"], n) for n in lk]


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _offsets(lengths):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = dict(case)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        s["x"] = _randn(gen, m, k, dtype=dt)
        s["w"] = _randn(gen, n, k, dtype=dt, scale=k ** -0.5)
        s["b"] = _randn(gen, n, dtype=dt, scale=0.2) if case["bias"] else None
        s["r"] = _randn(gen, m, n, dtype=dt) if case["residual"] else None
        if case["grad"]:
            s["dy"] = _randn(gen, m, n, dtype=dt)
            s["pre"] = None
            if case["act"] != "none":         # what the forward pass kept
                s["pre"] = torch.matmul(s["x"], s["w"].t())
                if case["bias"]:
                    s["pre"] = s["pre"] + s["b"]
        return s
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["op"] == "rope":
        t, half = case["rows"], case["rot"] // 2
        fused = _randn(gen, t, (hq + 2 * hk) * d, dtype=dt)          # one projection: queries, keys, values
        s["q"] = fused[:, :hq * d].unflatten(1, (hq, d))
        s["k"] = fused[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
        s["qw"] = 1.0 + 0.1 * _randn(gen, d) if case["weight"] else None
        s["kw"] = 1.0 + 0.1 * _randn(gen, d) if case["weight"] else None
        places = 1200
        angle = torch.arange(places, device="cuda")[:, None] * 100.0 ** (-torch.arange(half, device="cuda") / half)
        s["cos"], s["sin"] = angle.cos(), angle.sin()
        s["pos"] = torch.randint(0, places, (t,), generator=gen, device="cuda", dtype=torch.int32)
        if case["grad"]:
            s["dq"], s["dk"] = _randn(gen, t, hq, d, dtype=dt), _randn(gen, t, hk, d, dtype=dt)
        return s
    lq, lk, prefix = _lengths(case)
    docs = case["docs"]
    tq = sum(lq)
    s["cu_q"] = _offsets(lq)
    if case["cache"]:                          # a cache with room for every stream's longest
        s["cu_k"] = _offsets([case["max_k"]] * docs)
        s["k_len"] = torch.tensor(lk, dtype=torch.int32, device="cuda")
        tk = docs * case["max_k"]
    else:
        s["cu_k"], s["k_len"], tk = _offsets(lk), None, sum(lk)
    s["prefix_len"] = torch.tensor(prefix, dtype=torch.int32, device="cuda") if case["prefix"] else None
    # normalised queries and keys, as qk_norm_rope leaves them
    s["q"] = _randn(gen, tq, hq, d, dtype=dt)
    s["k"] = _randn(gen, tk, hk, d, dtype=dt)
    s["v"] = _randn(gen, tk, hk, d, dtype=dt)
    s["slopes"] = torch.exp2(-8.0 * (torch.arange(hq, device="cuda") + 1) / hq) if case["bias"] else None
    s["scale"] = d ** -0.5
    if case["grad"]:
        s["do"] = _randn(gen, tq, hq, d, dtype=dt)
        o, lse = _attention_plain(s)           # what the forward pass kept
        s["o"], s["lse"] = o, lse
    return s


# ----------------------------------------------------------------------------------------------------------------- #
# The plain forms: elementary operations in 32 bits, rounded once
# ----------------------------------------------------------------------------------------------------------------- #
def _erf_gelu_parts(z):
    phi = 0.5 * (1.0 + torch.erf(z * 2.0 ** -0.5))
    return phi, torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return z * _erf_gelu_parts(z)[0]
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    phi, density = _erf_gelu_parts(z)
    return phi + z * density


def _linear_plain(s):
    dt = s["x"].dtype
    z = torch.matmul(s["x"].float(), s["w"].float().t())
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return (y.to(dt), z.to(dt)) if s["save"] else y.to(dt)


def _linear_grad_plain(s):
    dt = s["x"].dtype
    dz = s["dy"].float()
    if s["pre"] is not None:
        dz = dz * _act_slope(s["pre"].float(), s["act"])
    dx = torch.matmul(dz, s["w"].float())
    dw = torch.matmul(dz.t(), s["x"].float())
    return dx.to(dt), dw.to(dt), dz.sum(0).to(dt) if s["bias"] else None


def _turn(x, cos, sin, interleaved):
    """Rotates the pairs of the first 2 * cos.shape[-1] values of each head."""
    h = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * h:]], -1)


def _angles(s, dtype):
    at = s["pos"].long()
    return s["cos"][at].to(dtype)[:, None], s["sin"][at].to(dtype)[:, None]


def _norm_turn(x, w, cos, sin, interleaved):
    f = x.float()
    n = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)
    if w is not None:
        n = n * w
    return _turn(n, cos, sin, interleaved).to(x.dtype)


def _norm_turn_grad(dy, x, w, cos, sin, interleaved):
    f = x.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)
    g = _turn(dy.float(), cos, -sin, interleaved)          # the rotation's transpose
    n = f * r
    dw = (g * n).sum((0, 1)) if w is not None else None
    if w is not None:
        g = g * w
    return (r * (g - n * (g * n).mean(-1, keepdim=True))).to(x.dtype), dw


def _padded(s):
    """Index tensors from packed rows to [documents, longest] and back."""
    dev, mq, mk = s["q"].device, s["max_q"], s["max_k"]
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    lq, lk = cq[1:] - cq[:-1], ck[1:] - ck[:-1]
    if s["k_len"] is not None:
        lk = s["k_len"].long()
    iq, ik = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    rows = (cq[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)
    cols = (ck[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    has_q, has_k = iq < lq[:, None], ik < lk[:, None]
    place = iq + (lk - lq)[:, None]                        # a query's place among its document's keys
    allowed = has_q[:, :, None] & has_k[:, None, :]
    if s["causal"]:
        seen = ik <= place[:, :, None]
        if s["prefix_len"] is not None:
            seen = seen | (ik < s["prefix_len"].long()[:, None, None])
        allowed = allowed & seen
    far = (place[:, :, None] - ik).abs().float()
    return rows, cols, has_q, has_k, allowed, far


def _scores(s, rows, cols, has_k, allowed, far):
    """Masked scores [documents, key heads, group, queries, keys], the capped ones before the bias, and the operands."""
    n, mq, mk = rows.shape[0], rows.shape[1], cols.shape[1]
    hk, d = s["k"].shape[1], s["q"].shape[2]
    g = s["q"].shape[1] // hk
    q = s["q"][rows].float().view(n, mq, hk, g, d).permute(0, 2, 3, 1, 4)
    k = s["k"][cols].float().permute(0, 2, 1, 3)
    v = torch.where(has_k[:, :, None, None], s["v"][cols].float(), 0.0).permute(0, 2, 1, 3)
    x = torch.matmul(q.reshape(n, hk, g * mq, d), k.transpose(-1, -2)).view(n, hk, g, mq, mk) * s["scale"]
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    capped = x
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, hk, g, 1, 1) * far[:, None, None]
    return torch.where(allowed[:, None, None], x, -math.inf), capped, q, k, v


def _unpad(x, at, cu):
    """Rows of x [documents, longest, ...] back in packed order."""
    t = torch.arange(at, device=x.device)
    doc = torch.searchsorted(cu, t.to(cu.dtype), right=True) - 1
    return x[doc, t - cu.long()[doc]]


def _attention_plain(s):
    rows, cols, has_q, has_k, allowed, far = _padded(s)
    x, _, q, k, v = _scores(s, rows, cols, has_k, allowed, far)
    n, hk, g, mq, mk = x.shape
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p.view(n, hk, g * mq, mk), v).view(n, hk, g, mq, -1)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, mq, hk * g, -1)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(n, mq, hk * g)
    tq = s["q"].shape[0]
    return _unpad(o, tq, s["cu_q"]).to(s["q"].dtype), _unpad(lse, tq, s["cu_q"]).t().contiguous()


def _attention_grad_plain(s):
    rows, cols, has_q, has_k, allowed, far = _padded(s)
    x, capped, q, k, v = _scores(s, rows, cols, has_k, allowed, far)
    n, hk, g, mq, mk = x.shape
    d = q.shape[-1]
    heads = lambda t: t[rows].float().view(n, mq, hk, g, -1).permute(0, 2, 3, 1, 4)  # noqa: E731
    do = torch.where(has_q[:, None, None, :, None], heads(s["do"]), 0.0)
    o = heads(s["o"])
    lse = s["lse"].t()[rows].view(n, mq, hk, g).permute(0, 2, 3, 1)[..., None]
    p = torch.where(allowed[:, None, None], torch.exp(x - lse), 0.0)
    flat = lambda t: t.reshape(n, hk, g * mq, -1)  # noqa: E731
    dv = torch.matmul(flat(p).transpose(-1, -2), flat(do))
    dp = torch.matmul(flat(do), v.transpose(-1, -2)).view_as(p)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    if s["softcap"]:
        ds = ds * (1.0 - (capped / s["softcap"]) ** 2)
    ds = ds * s["scale"]
    dq = torch.matmul(flat(ds), k).view(n, hk, g, mq, d).permute(0, 3, 1, 2, 4).reshape(n, mq, hk * g, d)
    dk = torch.matmul(flat(ds).transpose(-1, -2), flat(q))
    tq, tk, dt = s["q"].shape[0], s["k"].shape[0], s["q"].dtype
    return (_unpad(dq, tq, s["cu_q"]).to(dt), _unpad(dk.permute(0, 2, 1, 3), tk, s["cu_k"]).to(dt),
            _unpad(dv.permute(0, 2, 1, 3), tk, s["cu_k"]).to(dt))


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "linear":
        return _linear_grad_plain(s) if s["grad"] else _linear_plain(s)
    if s["op"] == "rope":
        cos, sin = _angles(s, torch.float32)
        if s["grad"]:
            dq, dqw = _norm_turn_grad(s["dq"], s["q"], s["qw"], cos, sin, s["interleaved"])
            dk, dkw = _norm_turn_grad(s["dk"], s["k"], s["kw"], cos, sin, s["interleaved"])
            return dq, dk, dqw, dkw
        return (_norm_turn(s["q"], s["qw"], cos, sin, s["interleaved"]),
                _norm_turn(s["k"], s["kw"], cos, sin, s["interleaved"]))
    return _attention_grad_plain(s) if s["grad"] else _attention_plain(s)


def _run_own(s):
    from promptmoge_b200 import tokens
    if s["op"] == "linear":
        if s["grad"]:
            return tokens.linear_grad(s["dy"], s["x"], s["w"], pre=s["pre"], activation=s["act"],
                                      bias_grad=s["bias"])
        return tokens.linear(s["x"], s["w"], s["b"], activation=s["act"], residual=s["r"], save_pre=s["save"])
    if s["op"] == "rope":
        if s["grad"]:
            return tokens.qk_norm_rope_grad(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"],
                                            s["pos"], eps=1e-6, interleaved=s["interleaved"])
        return tokens.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"], eps=1e-6,
                                   interleaved=s["interleaved"])
    mask = dict(scale=s["scale"], causal=s["causal"], prefix=s["prefix_len"], softcap=s["softcap"],
                slopes=s["slopes"], k_len=s["k_len"])
    packing = (s["cu_q"], s["cu_k"], s["max_q"], s["max_k"])
    if s["grad"]:
        return tokens.attention_grad(s["do"], s["o"], s["lse"], s["q"], s["k"], s["v"], *packing, **mask)
    return tokens.attention(s["q"], s["k"], s["v"], *packing, **mask)


# ----------------------------------------------------------------------------------------------------------------- #
# What a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------- #
def _pairs(case):
    """Query-key pairs that the masks let through, over all documents, for one head."""
    total = 0
    for lq, lk, prefix in zip(*_lengths(case)):
        if not case["causal"]:
            total += lq * lk
        else:
            seen = np.clip(np.arange(lq) + (lk - lq) + 1, 0, lk)
            total += int(np.maximum(seen, prefix).sum())
    return total


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        if case["grad"]:
            kept = m * n if case["act"] != "none" else 0
            return {"bytes": size * (m * n + kept + 2 * m * k + 2 * n * k + n), "flops": 4 * m * n * k}
        outs = 1 + int(case["residual"]) + int(case["save"])
        return {"bytes": size * (m * k + n * k + n * int(case["bias"]) + outs * m * n), "flops": 2 * m * n * k}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["op"] == "rope":
        t = case["rows"]
        values = t * (hq + hk) * d
        table = min(t, 1200) * case["rot"] * 4 + 4 * t
        return {"bytes": size * values * (3 if case["grad"] else 2) + table, "flops": values * (16 if case["grad"] else 8)}
    lq, lk, _ = _lengths(case)
    tq, tk, pairs = sum(lq), sum(lk), _pairs(case)
    if case["grad"]:
        return {"bytes": size * d * (4 * tq * hq + 4 * tk * hk) + 4 * tq * hq, "flops": 10 * d * hq * pairs}
    return {"bytes": size * d * (2 * tq * hq + 2 * tk * hk) + 4 * tq * hq, "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------------------------------------------------- #
# The definitions in 64 bits, document by document
# ----------------------------------------------------------------------------------------------------------------- #
def _exact_linear(s):
    x, w = s["x"].double(), s["w"].double()
    act = s["act"]
    if s["grad"]:
        g = s["dy"].double()
        if act != "none":
            z = s["pre"].double().requires_grad_(True)
            y = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](z)
            g, = torch.autograd.grad(y, z, g)
        return g @ w, g.t() @ x, g.sum(0) if s["bias"] else None
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].double()
    y = z if act == "none" else {"relu": torch.relu, "silu": torch.nn.functional.silu,
                                 "gelu": torch.nn.functional.gelu}[act](z)
    if s["r"] is not None:
        y = y + s["r"].double()
    return (y, z) if s["save"] else y


def _exact_rope(s):
    def one(x, w):
        n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        n = n if w is None else n * w
        h = s["rot"] // 2
        at = s["pos"].long()
        turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]
        head = n[..., :2 * h]
        pair = head.unflatten(-1, (h, 2)) if s["interleaved"] else head.unflatten(-1, (2, h)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, n[..., 2 * h:]], -1)

    outs, grads = [], []
    for x, w, dy in ((s["q"], s["qw"], s.get("dq")), (s["k"], s["kw"], s.get("dk"))):
        x = x.double().requires_grad_(True)
        w = None if w is None else w.double().requires_grad_(True)
        y = one(x, w)
        outs.append(y.detach())
        if s["grad"]:
            grads.append(torch.autograd.grad(y, [x] if w is None else [x, w], dy.double()))
    if not s["grad"]:
        return tuple(outs)
    (dq, *dqw), (dk, *dkw) = grads
    return dq, dk, dqw[0] if dqw else None, dkw[0] if dkw else None


def _exact_attention(s):
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    kl = s["k_len"].tolist() if s["k_len"] is not None else [b - a for a, b in zip(ck, ck[1:])]
    pre = s["prefix_len"].tolist() if s["prefix_len"] is not None else [0] * len(kl)
    q, k, v = (s[n].double() for n in "qkv")
    hq, hk = q.shape[1], k.shape[1]
    o, lse = torch.zeros_like(q), torch.full((hq, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for n in range(len(kl)):
        a, b, c, e = cq[n], cq[n + 1], ck[n], ck[n] + kl[n]
        if a == b or c == e:
            continue
        place = torch.arange(b - a, device=q.device)[:, None] + (kl[n] - (b - a))
        j = torch.arange(kl[n], device=q.device)[None]
        ok = torch.ones(b - a, kl[n], dtype=torch.bool, device=q.device)
        if s["causal"]:
            ok = (j <= place) | (j < pre[n])
        for h in range(hq):
            g = h // (hq // hk)
            qs, ks, vs = (t.detach().requires_grad_(s["grad"]) for t in (q[a:b, h], k[c:e, g], v[c:e, g]))
            x = qs @ ks.t() * s["scale"]
            if s["softcap"]:
                x = s["softcap"] * torch.tanh(x / s["softcap"])
            if s["slopes"] is not None:
                x = x - s["slopes"][h].double() * (place - j).abs()
            x = x.masked_fill(~ok, -math.inf)
            l = torch.logsumexp(x, -1, keepdim=True)
            p = torch.where(ok, torch.exp(x - torch.where(l == -math.inf, 0.0, l)), 0.0)
            y = p @ vs
            o[a:b, h], lse[h, a:b] = y.detach(), l.detach()[:, 0]
            if s["grad"]:
                gq, gk, gv = torch.autograd.grad(y, [qs, ks, vs], s["do"][a:b, h].double())
                dq[a:b, h] = gq
                dk[c:e, g] += gk
                dv[c:e, g] += gv
    return (dq, dk, dv) if s["grad"] else (o, lse)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s)
    return _exact_rope(s) if case["op"] == "rope" else _exact_attention(s)
