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


def grad_reference(q, k, v, do, cu_q, cu_k, scale, u, causal=False, prefix=None, softcap=0.0, slopes=None, k_len=None):
    """Gradients (dq, dk, dv) by the formula, in float64, and how far a computation may be off that rounds P, dS, o and
    its results to unit roundoff u and carries scores with relative error e in each probability: a list of three
    bounds of the same shapes."""
    cq, ck = cu_q.tolist(), cu_k.tolist()
    kl = k_len.tolist() if k_len is not None else [b - a for a, b in zip(ck, ck[1:])]
    pre = prefix.tolist() if prefix is not None else [0] * len(kl)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    g = q.shape[1] // k.shape[1]
    grads, bounds = ([torch.zeros_like(t) for t in (q, k, v)] for _ in range(2))
    for n in range(len(kl)):
        a, b, c, f = cq[n], cq[n + 1], ck[n], ck[n] + kl[n]
        if a == b or c == f:
            continue
        place = torch.arange(b - a, device=q.device)[:, None] + (kl[n] - (b - a))
        j = torch.arange(kl[n], device=q.device)[None]
        ok = (j <= place) | (j < pre[n]) if causal else torch.ones(b - a, kl[n], dtype=torch.bool, device=q.device)
        qs, ds_ = (t[a:b].transpose(0, 1) for t in (q, do))
        kr, vr = (t[c:f].transpose(0, 1).repeat_interleave(g, 0) for t in (k, v))
        x = qs @ kr.transpose(1, 2) * scale
        S = float(qs.norm(dim=-1).max() * kr.norm(dim=-1).max()) * scale
        slope = torch.ones_like(x)
        if softcap:
            t = torch.tanh(x / softcap)
            x, slope = softcap * t, 1 - t * t
        if slopes is not None:
            x = x - slopes.double()[:, None, None] * (place - j).abs()
            S += float(slopes.max()) * max(b - a, kl[n])
        e = 2.0 ** -18 * (1 + S)
        x = x.masked_fill(~ok, -math.inf)
        top = torch.logsumexp(x, -1, keepdim=True)
        p = torch.where(ok, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
        o = p @ vr
        dp = ds_ @ vr.transpose(1, 2)
        delta = (ds_ * o).sum(-1, keepdim=True)
        dS = p * (dp - delta) * slope
        size = ds_.abs() @ vr.abs().transpose(1, 2)
        off = (u + e) * dS.abs() + p * (2.0 ** -18 * size + (u + 2.0 ** -20) * (ds_ * o).abs().sum(-1, keepdim=True))
        off = off + 2.0 ** -18 * p * (dp - delta).abs()          # the cap's slope, 1 - t^2 of a rounded t
        sums = lambda y: y.unflatten(0, (-1, g)).sum(1).transpose(0, 1)  # noqa: E731
        grads[0][a:b] = (dS @ kr * scale).transpose(0, 1)
        grads[1][c:f] += sums(dS.transpose(1, 2) @ qs * scale)
        grads[2][c:f] += sums(p.transpose(1, 2) @ ds_)
        bounds[0][a:b] = (off @ kr.abs() * scale).transpose(0, 1)
        bounds[1][c:f] += sums(off.transpose(1, 2) @ qs.abs() * scale)
        bounds[2][c:f] += (u + e) * sums(p.transpose(1, 2) @ ds_.abs())
    return grads, [t * 1.01 + u * y.abs() + 1e-7 for t, y in zip(bounds, grads)]
