"""The float64 attention that the GPU tests compare with: its gradient formula against autograd and against differences,
on the CPU."""
import pytest
import torch

from attention_reference import grad_reference, offsets, reference

MASKS = [dict(), dict(causal=True), dict(causal=True, prefix=True), dict(softcap=5.0),
         dict(causal=True, prefix=True, softcap=4.0, slopes=True)]


def _case(mask, seed=0):
    gen = torch.Generator().manual_seed(seed)
    lq, lk = [5, 0, 3, 9], [5, 4, 8, 2]
    q, k, v, do = (torch.randn(n, h, 8, generator=gen, dtype=torch.float64)
                   for n, h in ((17, 4), (19, 2), (19, 2), (17, 4)))
    kw = {n: x for n, x in mask.items() if n in ("causal", "softcap")}
    if mask.get("prefix"):
        kw["prefix"] = torch.tensor([2, 0, 8, 1], dtype=torch.int32)
    if mask.get("slopes"):
        kw["slopes"] = torch.tensor([0.5, 0.25, 0.1, 0.0], dtype=torch.float64)
    return q, k, v, do, offsets(lq, "cpu"), offsets(lk, "cpu"), kw


@pytest.mark.parametrize("mask", MASKS)
def test_gradient_formula(mask):
    q, k, v, do, cq, ck, kw = _case(mask)
    want = reference(q, k, v, cq, ck, 0.35, do=do, **kw)[3:]
    got, _ = grad_reference(q, k, v, do, cq, ck, 0.35, 0.0, **kw)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)
    base = [q, k, v]
    for i in range(3):
        d, h = got[i], 1e-5
        ends = []
        for sign in (1, -1):
            x = list(base)
            x[i] = base[i] + sign * h * d
            ends.append((reference(*x, cq, ck, 0.35, **kw)[0] * do).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) / d.square().sum() - 1) < 1e-6
