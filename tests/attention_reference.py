"""Attention over packed documents in float64, document by document: the definition the kernels are tested against."""
import math

import torch


def offsets(lengths, device="cuda"):
    return torch.tensor([0] + list(torch.tensor(lengths, dtype=torch.int64).cumsum(0)), dtype=torch.int32, device=device)


def reference(q, k, v, cu_q, cu_k, scale, causal=False, prefix=None, softcap=0.0, slopes=None, k_len=None, do=None):
    """(o, lse) and, with do, the gradients (dq, dk, dv); also sum p |v| per output, for tolerances."""
    cq, ck = cu_q.tolist(), cu_k.tolist()
    kl = k_len.tolist() if k_len is not None else [b - a for a, b in zip(ck, ck[1:])]
    pre = prefix.tolist() if prefix is not None else [0] * len(kl)
    q, k, v = q.double(), k.double(), v.double()
    hq, hk = q.shape[1], k.shape[1]
    o, mass = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((hq, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    for n in range(len(kl)):
        a, b, c, e = cq[n], cq[n + 1], ck[n], ck[n] + kl[n]
        if a == b or c == e:
            continue
        place = torch.arange(b - a, device=q.device)[:, None] + (kl[n] - (b - a))
        j = torch.arange(kl[n], device=q.device)[None]
        ok = (j <= place) | (j < pre[n]) if causal else torch.ones(b - a, kl[n], dtype=torch.bool, device=q.device)
        qs = q[a:b].transpose(0, 1).clone().requires_grad_(True)
        ks = k[c:e].transpose(0, 1).clone().requires_grad_(True)
        vs = v[c:e].transpose(0, 1).clone().requires_grad_(True)
        kr, vr = (t.repeat_interleave(hq // hk, 0) for t in (ks, vs))
        x = qs @ kr.transpose(1, 2) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        if slopes is not None:
            x = x - slopes.double()[:, None, None] * (place - j).abs()
        x = x.masked_fill(~ok, -math.inf)
        top = torch.logsumexp(x, -1, keepdim=True)
        p = torch.where(ok, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
        y = p @ vr
        o[a:b], lse[:, a:b] = y.detach().transpose(0, 1), top.detach()[..., 0]
        mass[a:b] = (p.detach() @ vr.detach().abs()).transpose(0, 1)
        if do is not None:
            g = torch.autograd.grad(y, [qs, ks, vs], do[a:b].double().transpose(0, 1))
            grads[0][a:b] = g[0].transpose(0, 1)
            grads[1][c:e] += g[1].transpose(0, 1)
            grads[2][c:e] += g[2].transpose(0, 1)
    return (o, lse, mass) if do is None else (o, lse, mass, *grads)
