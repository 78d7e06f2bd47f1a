"""Attention over packed documents against float64.

Tolerances.  u is the operands' unit roundoff.  The output is rounded once (u |o|); probabilities are rounded once to
the operands' type (u sum p|v|); scores carry fp32 error, at most 2^-19 times the largest score's size S a row can meet
(|q||k| scale, plus the distance bias), which moves each probability by that share: in all u |o| + (u + 2^-18 (1 + S))
sum p|v|, and 2^-18 (1 + S) for the log sum."""
import math

import pytest
import torch

from attention_reference import offsets, reference

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(lq, lk, hq, hk, d, dtype, seed=0, slopes=False, room=None):
    gen = torch.Generator(device="cuda").manual_seed(seed + sum(lq) + 3 * sum(lk) + d)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    tk = sum(room or lk)
    sl = torch.exp2(-8.0 * (torch.arange(hq, device="cuda") + 1) / hq) if slopes else None
    return rand(sum(lq), hq, d), rand(tk, hk, d), rand(tk, hk, d), offsets(lq), offsets(room or lk), sl


def near(got, lse, ref, scale, q, k, slopes, longest, dtype):
    o, want_lse, mass = ref[:3]
    S = scale * float(q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max())
    if slopes is not None:
        S += float(slopes.max()) * longest
    u, e = U[dtype], 2.0 ** -18 * (1 + S)
    assert torch.equal(torch.isneginf(lse), torch.isneginf(want_lse))
    fin = ~torch.isneginf(want_lse)
    assert ((lse.double() - want_lse)[fin].abs() <= e).all()
    err = (got.double() - o).abs() - (u * o.abs() + (u + e) * mass + 1e-7)
    assert (err <= 0).all(), float(err.max())


LENGTHS = [([1], [1]), ([5], [5]), ([128], [128]), ([129, 0, 127], [129, 0, 127]), ([300, 1, 64], [300, 1, 64]),
           ([257, 40], [385, 300]), ([100], [30]), ([0, 0, 33], [5, 0, 700]), ([700], [700]), ([1200, 900], [1200, 900])]
MASKS = [dict(), dict(causal=True), dict(causal=True, prefix=True), dict(softcap=20.0), dict(slopes=True),
         dict(causal=True, prefix=True, softcap=30.0, slopes=True)]


def options(mask, lk, slopes):
    kw = {n: v for n, v in mask.items() if n in ("causal", "softcap")}
    if mask.get("prefix"):
        kw["prefix"] = torch.tensor([min(n, 7 + 90 * i) for i, n in enumerate(lk)], dtype=torch.int32, device="cuda")
    if mask.get("slopes"):
        kw["slopes"] = slopes
    return kw


@pytest.mark.parametrize("lq,lk", LENGTHS)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("hq,hk,d,dtype", [(4, 4, 64, torch.bfloat16), (4, 2, 128, torch.float16),
                                           (3, 1, 40, torch.float16), (8, 1, 104, torch.bfloat16)])
def test_attention_equals_float64(lq, lk, mask, hq, hk, d, dtype):
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, sl = make(lq, lk, hq, hk, d, dtype, slopes=True)
    kw = options(mask, lk, sl)
    scale = d ** -0.5
    o, lse = tokens.attention(q, k, v, cq, ck, max(lq), max(lk), scale=scale, **kw)
    tokens.check()
    near(o, lse, reference(q, k, v, cq, ck, scale, **kw), scale, q, k, kw.get("slopes"), max(lq + lk), dtype)


@pytest.mark.parametrize("max_q,hq,hk", [(1, 1, 1), (1, 16, 4), (1, 16, 1), (3, 8, 2), (16, 2, 2), (4, 16, 4)])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (24, torch.float16), (96, torch.bfloat16)])
@pytest.mark.parametrize("mask", MASKS)
def test_few_rows_over_a_cache(max_q, hq, hk, d, dtype, mask):
    """Caches with spare room, used parts of every length; what lies in the room is never a number."""
    from promptmoge_b200 import tokens
    lk = [1, 16, 31, 33, 260, 0, 1025, 5000, 4096]
    lq = [max_q if i % 3 else max(0, max_q - 1) for i in range(len(lk))]
    room = [n + 70 for n in lk]
    q, k, v, cq, ck, sl = make(lq, lk, hq, hk, d, dtype, slopes=True, room=room)
    used = torch.tensor(lk, dtype=torch.int32, device="cuda")
    for n, c in zip(lk, ck.tolist()):
        k[c + n:c + n + 70] = float("nan")
        v[c + n:c + n + 70] = float("inf")
    kw = options(mask, lk, sl)
    o, lse = tokens.attention(q, k, v, cq, ck, max_q, max(room), k_len=used, **kw)
    tokens.check()
    clean_k, clean_v = torch.nan_to_num(k, nan=0.0), torch.where(torch.isfinite(v), v, 0.0)
    near(o, lse, reference(q, clean_k, clean_v, cq, ck, d ** -0.5, k_len=used, **kw), d ** -0.5, q, clean_k,
         kw.get("slopes"), 5000, dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_documents_do_not_reach_each_other(d, causal):
    """NaN and infinities in one document's queries, keys and values leave the others' results as they are."""
    from promptmoge_b200 import tokens
    lq = [130, 200, 77, 256, 20]
    q, k, v, cq, ck, _ = make(lq, lq, 4, 2, d, torch.bfloat16)
    want, want_lse = tokens.attention(q, k, v, cq, ck, 256, 256, causal=causal)
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        t[330:407] = bad
    got, lse = tokens.attention(q, k, v, cq, ck, 256, 256, causal=causal)
    keep = torch.ones(sum(lq), dtype=torch.bool, device="cuda")
    keep[330:407] = False
    assert torch.equal(got[keep], want[keep]) and torch.equal(lse[:, keep], want_lse[:, keep])


@pytest.mark.parametrize("max_q,lk", [(1, 3000), (300, 300)])
def test_large_scores_and_infinities(max_q, lk):
    """A maximum that moves by hundreds over the keys; a key of -inf score takes no part."""
    from promptmoge_b200 import tokens
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v, cq, ck, _ = make([max_q], [lk], 2, 1, 64, dtype)
        k = (k.float() * torch.linspace(0.2, 6, lk, device="cuda")[:, None, None]).to(dtype)
        q = (q.float() * 5).to(dtype)
        o, lse = tokens.attention(q, k, v, cq, ck, max_q, lk, scale=0.125)
        near(o, lse, reference(q, k, v, cq, ck, 0.125), 0.125, q, k, None, lk, dtype)
    q[:, :, 0] = 1.0
    k[5, :, :] = 0.0
    k[5, :, 0] = -math.inf
    o, lse = tokens.attention(q, k, v, cq, ck, max_q, lk, scale=0.125)
    keep = torch.arange(lk, device="cuda") != 5
    ref = reference(q, k[keep], v[keep], cq, offsets([lk - 1]), 0.125)
    near(o, lse, ref, 0.125, q, k[keep], None, lk, dtype)


def test_strided_heads_and_output():
    """Queries, keys and values in place in one projection, heads before tokens, output inside a larger tensor."""
    from promptmoge_b200 import tokens
    gen = torch.Generator(device="cuda").manual_seed(0)
    fused = torch.randn(400, 6 * 64 + 16, generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = (fused[:, 8 + s * 64:8 + e * 64].unflatten(1, (e - s, 64)) for s, e in ((0, 4), (4, 5), (5, 6)))
    cu = offsets([250, 150])
    big = torch.zeros(400, 5, 72, dtype=torch.bfloat16, device="cuda")
    o, lse = tokens.attention(q, k, v, cu, cu, 250, 250, causal=True, out=big[:, :4, :64])
    near(o, lse, reference(q, k, v, cu, cu, 0.125, causal=True), 0.125, q, k, None, 250, torch.bfloat16)
    assert not big[:, 4].any() and not big[:, :, 64:].any()
    qt, kt, vt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    o2, lse2 = tokens.attention(qt, kt, vt, cu, cu, 250, 250, causal=True)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)


def test_many_short_documents():
    from promptmoge_b200 import tokens
    lens = [(7 * i) % 41 for i in range(1500)]
    q, k, v, cq, ck, _ = make(lens, lens, 2, 2, 64, torch.float16)
    o, lse = tokens.attention(q, k, v, cq, ck, 40, 40, causal=True)
    near(o, lse, reference(q, k, v, cq, ck, 0.125, causal=True), 0.125, q, k, None, 40, torch.float16)


def test_without_tokens_and_repeats():
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([0], [40], 4, 2, 64, torch.float16)
    o, lse = tokens.attention(q, k, v, cq, ck, 0, 40)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    q, k, v, cq, ck, _ = make([50], [0], 4, 2, 64, torch.float16)
    o, lse = tokens.attention(q, k, v, cq, ck, 50, 0)
    assert not o.any() and torch.isneginf(lse).all()
    q, k, v, cq, ck, _ = make([2], [9000], 4, 2, 64, torch.float16)
    a, b = (tokens.attention(q, k, v, cq, ck, 2, 9000) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_document_longer_than_max_q_is_reported():
    from promptmoge_b200 import tokens
    from promptmoge_b200._lib import PmgError
    q, k, v, cq, ck, _ = make([3], [40], 4, 4, 64, torch.float16)
    tokens.attention(q, k, v, cq, ck, 1, 40)
    with pytest.raises(PmgError):
        tokens.check()


def test_refusals():
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, sl = make([30], [40], 4, 2, 64, torch.float16, slopes=True)
    base = dict(q=q, k=k, v=v, cu_q=cq, cu_k=ck, max_q=30, max_k=40)
    for change in (dict(q=q.cpu()), dict(k=k[:, :, :32]), dict(v=v[:20]), dict(k=k[:, :1].expand(40, 3, 64), v=k[:, :1].expand(40, 3, 64)),
                   dict(cu_q=cq[:1].repeat(3)), dict(scale=0.0), dict(scale=float("inf")), dict(softcap=-1.0),
                   dict(slopes=sl[:2]), dict(prefix=cq[:1]), dict(max_q=-1), dict(q=q[:, :, :60], k=k[:, :, :60], v=v[:, :, :60]),
                   dict(k_len=cq), dict(q=q.flatten()[4:4 + 29 * 256].view(29, 4, 64), cu_q=offsets([29]))):
        with pytest.raises(ValueError):
            tokens.attention(**(base | change))
    for change in (dict(q=q.float()), dict(k=k.bfloat16()), dict(cu_q=cq.long()), dict(slopes=sl.double())):
        with pytest.raises(TypeError):
            tokens.attention(**(base | change))
