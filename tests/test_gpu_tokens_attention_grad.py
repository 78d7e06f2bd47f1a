"""Gradients of attention over packed documents against the formula in float64.

Tolerances (attention_reference.grad_reference): P, dS and the results are rounded to the operands' unit roundoff u, o
(which delta is formed from) was; scores carry fp32 error as in the forward test; sums are fp32."""
import pytest
import torch

from attention_reference import grad_reference, offsets, reference
from test_gpu_tokens_attention import LENGTHS, MASKS, U, make, options

pytestmark = pytest.mark.gpu


def run(lq, lk, hq, hk, d, dtype, mask, scale=None, room=None, grow=1.0):
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, sl = make(lq, lk, hq, hk, d, dtype, slopes=True, room=room)
    gen = torch.Generator(device="cuda").manual_seed(9)
    do = (torch.randn(q.shape, generator=gen, device="cuda") * grow).to(dtype)
    kw = options(mask, lk, sl)
    if room is not None:
        kw["k_len"] = torch.tensor(lk, dtype=torch.int32, device="cuda")
    scale = d ** -0.5 if scale is None else scale
    most = (max(lq), max(room or lk))
    o, lse = tokens.attention(q, k, v, cq, ck, *most, scale=scale, **kw)
    got = tokens.attention_grad(do, o, lse, q, k, v, cq, ck, *most, scale=scale, **kw)
    tokens.check()
    want, bounds = grad_reference(q, k, v, do, cq, ck, scale, U[dtype], **kw)
    return got, want, bounds


def close(got, want, bounds):
    for name, g, w, b in zip(("dq", "dk", "dv"), got, want, bounds):
        err = (g.double() - w).abs() - b
        assert (err <= 0).all(), (name, float(err.max()))


@pytest.mark.parametrize("lq,lk", LENGTHS)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("hq,hk,d,dtype", [(4, 4, 64, torch.bfloat16), (4, 2, 128, torch.float16),
                                           (3, 1, 40, torch.float16), (8, 1, 104, torch.bfloat16)])
def test_gradients_equal_float64(lq, lk, mask, hq, hk, d, dtype):
    close(*run(lq, lk, hq, hk, d, dtype, mask))


@pytest.mark.parametrize("grow", [2.0 ** -11, 2.0 ** 6])
def test_small_and_large_gradients_in_fp16(grow):
    """Loss scales: gradients whose dS would be subnormal, or overflow, in fp16."""
    got, want, bounds = run([300, 40], [300, 40], 2, 1, 64, torch.float16, dict(causal=True), grow=grow)
    bounds = [b + 2.0 ** -25 for b in bounds]            # fp16's own spacing near zero
    close(got, want, bounds)


def test_rows_behind_a_cache_get_zeros():
    lk, room = [30, 0, 129], [100, 40, 300]
    got, want, bounds = run([30, 5, 7], lk, 4, 2, 64, torch.bfloat16, dict(causal=True), room=room)
    close(got, want, bounds)
    assert not got[1][30:140].any() and not got[2][269:].any()


@pytest.mark.parametrize("d", [64, 128])
def test_documents_do_not_reach_each_other(d):
    from promptmoge_b200 import tokens
    lens = [130, 200, 77, 256, 20]
    q, k, v, cq, ck, _ = make(lens, lens, 4, 2, d, torch.bfloat16)
    do = torch.randn_like(q)

    def grads():
        o, lse = tokens.attention(q, k, v, cq, ck, 256, 256)
        return tokens.attention_grad(do, o, lse, q, k, v, cq, ck, 256, 256)
    want = grads()
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (do, float("nan"))):
        t[330:407] = bad
    got = grads()
    keep = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    keep[330:407] = False
    for a, b in zip(got, want):
        assert torch.equal(a[keep], b[keep])


def test_against_differences():
    """The float64 loss's slope along the computed gradients, by central differences."""
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, sl = make([70, 9], [70, 40], 4, 2, 32, torch.float16, slopes=True)
    do = torch.randn_like(q)
    kw = dict(causal=True, prefix=torch.tensor([10, 3], dtype=torch.int32, device="cuda"), softcap=3.0, slopes=sl)
    o, lse = tokens.attention(q, k, v, cq, ck, 70, 70, **kw)
    got = [t.double() for t in tokens.attention_grad(do, o, lse, q, k, v, cq, ck, 70, 70, **kw)]
    base = [t.double() for t in (q, k, v)]
    for i in range(3):
        h, ends = 1e-4 / got[i].norm(), []
        for sign in (1, -1):
            x = list(base)
            x[i] = base[i] + sign * h * got[i]
            ends.append((reference(*x, cq, ck, 32 ** -0.5, **kw)[0] * do.double()).sum())
        # fp16 roundings of P, dS, o and the result are below 2^-9 of the gradient's norm
        assert abs((ends[0] - ends[1]) / (2 * h) / got[i].square().sum() - 1) < 5e-3


def test_many_short_documents_and_repeats():
    from promptmoge_b200 import tokens
    lens = [(7 * i) % 41 for i in range(700)]
    close(*run(lens, lens, 2, 2, 64, torch.float16, dict(causal=True)))
    q, k, v, cq, ck, _ = make([600], [600], 8, 1, 64, torch.bfloat16)
    o, lse = tokens.attention(q, k, v, cq, ck, 600, 600)
    a, b = (tokens.attention_grad(q, o, lse, q, k, v, cq, ck, 600, 600) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_strided_heads():
    from promptmoge_b200 import tokens
    gen = torch.Generator(device="cuda").manual_seed(0)
    fused = torch.randn(400, 6 * 64 + 16, generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = (fused[:, 8 + s * 64:8 + e * 64].unflatten(1, (e - s, 64)) for s, e in ((0, 4), (4, 5), (5, 6)))
    cu = offsets([250, 150])
    do = torch.randn(4, 400, 64, device="cuda").to(torch.bfloat16).transpose(0, 1)
    o, lse = tokens.attention(q, k, v, cu, cu, 250, 250, causal=True)
    got = tokens.attention_grad(do, o, lse, q, k, v, cu, cu, 250, 250, causal=True)
    want = tokens.attention_grad(do.contiguous(), o, lse, q.contiguous(), k.contiguous(), v.contiguous(), cu, cu, 250,
                                 250, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_without_queries_or_keys():
    from promptmoge_b200 import tokens
    for lq, lk in (([0], [40]), ([50], [0])):
        q, k, v, cq, ck, _ = make(lq, lk, 4, 2, 64, torch.float16)
        o, lse = tokens.attention(q, k, v, cq, ck, 50, 40)
        g = tokens.attention_grad(q, o, lse, q, k, v, cq, ck, 50, 40)
        assert [t.shape for t in g] == [q.shape, k.shape, v.shape] and not any(t.any() for t in g)


def test_refusals():
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([30], [40], 4, 2, 64, torch.float16)
    o, lse = tokens.attention(q, k, v, cq, ck, 30, 40)
    base = dict(do=q, o=o, lse=lse, q=q, k=k, v=v, cu_q=cq, cu_k=ck, max_q=30, max_k=40)
    for change in (dict(do=q[:5]), dict(lse=lse.t()), dict(lse=lse[:, :5]), dict(o=o[..., :32]), dict(do=q.cpu()), dict(softcap=-1.0)):
        with pytest.raises(ValueError):
            tokens.attention_grad(**(base | change))
    for change in (dict(do=q.float()), dict(lse=lse.half())):
        with pytest.raises(TypeError):
            tokens.attention_grad(**(base | change))
