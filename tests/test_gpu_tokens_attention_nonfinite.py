"""Scores that are not finite, on keys that a row sees: the row shows it, whichever column the key falls on.

A NaN score, and one of +inf (whose softmax is inf - inf), make a row NaN, as the definition does; rows that do not see
the key keep their bits."""
import pytest
import torch

from attention_reference import offsets, reference
from test_gpu_tokens_attention import U, make, options

pytestmark = pytest.mark.gpu
MASKS = [dict(), dict(slopes=True), dict(softcap=20.0), dict(causal=True), dict(causal=True, slopes=True)]


@pytest.mark.parametrize("lq,hq,hk", [(100, 2, 1), (4, 4, 1)])            # by the tile; few rows
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (64, torch.float16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("mask", MASKS)
def test_a_score_that_is_not_finite_shows_in_its_rows(lq, hq, hk, d, dtype, mask):
    from promptmoge_b200 import tokens
    lk = 200
    q, k, v, cq, ck, sl = make([lq], [lk], hq, hk, d, dtype, slopes=True)
    kw = options(mask, [lk], sl)
    q[:, :, 0] = 1
    clean, clean_lse = tokens.attention(q, k, v, cq, ck, lq, lk, **kw)
    for j in [*range(104, 112), *range(130, 146), 196, 199]:
        for bad in (float("nan"), float("inf")):
            if bad == float("inf") and "softcap" in kw:
                continue                                   # the cap makes it finite
            x = k.clone()
            x[j] = 0
            x[j, :, 0] = bad
            o, lse = tokens.attention(q, x, v, cq, ck, lq, lk, **kw)
            sees = torch.arange(lq, device="cuda") + lk - lq >= j if mask.get("causal") else torch.ones(lq, dtype=torch.bool, device="cuda")
            assert torch.isnan(o[sees]).all(), (j, bad)
            assert not (torch.isfinite(lse[:, sees]) | torch.isneginf(lse[:, sees])).any(), (j, bad)
            assert torch.equal(o[~sees], clean[~sees]) and torch.equal(lse[:, ~sees], clean_lse[:, ~sees])


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("mask", MASKS)
def test_a_row_that_is_not_finite_shows_in_the_gradients(d, dtype, mask):
    """One query of NaN: its log sum is NaN, so its probabilities, and with them dV and dK of every key that it sees."""
    from promptmoge_b200 import tokens
    lq, lk = 70, 90
    q, k, v, cq, ck, sl = make([lq], [lk], 2, 1, d, dtype, slopes=True)
    kw = options(mask, [lk], sl)
    do = torch.randn_like(q)
    o, lse = tokens.attention(q, k, v, cq, ck, lq, lk, **kw)
    clean = tokens.attention_grad(do, o, lse, q, k, v, cq, ck, lq, lk, **kw)
    for i in range(32, 66):
        x, bad_lse = lse.clone(), float("nan")
        x[1, i] = bad_lse
        dq, dk, dv = tokens.attention_grad(do, o, x, q, k, v, cq, ck, lq, lk, **kw)
        seen = torch.arange(lk, device="cuda") <= i + lk - lq if mask.get("causal") else torch.ones(lk, dtype=torch.bool, device="cuda")
        assert torch.isnan(dv[seen]).all() and torch.isnan(dk[seen]).all() and torch.isnan(dq[i, 1]).all(), i
        assert torch.equal(dv[~seen], clean[2][~seen]) and torch.equal(dk[~seen], clean[1][~seen])
        rest = torch.arange(lq, device="cuda") != i
        assert torch.equal(dq[rest], clean[0][rest]) and torch.equal(dq[:, 0], clean[0][:, 0])


@pytest.mark.parametrize("lq,hq,hk", [(100, 2, 1), (4, 4, 1)])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("infinite", [64, 128, 200])
@pytest.mark.parametrize("slopes", [False, True])
def test_capped_scores_of_minus_infinity_count_as_the_cap(lq, hq, hk, d, dtype, infinite, slopes):
    """tanh takes -inf to -cap, a score like any other, also where a row's first keys have nothing else.  Tolerances as in
    the forward test, with the scores' size bounded by the cap (and the distances)."""
    from promptmoge_b200 import tokens
    lk, cap = 200, 1.0
    q, k, v, cq, ck, sl = make([lq], [lk], hq, hk, d, dtype, slopes=True)
    q[:, :, 0] = 1
    k[:infinite] = 0
    k[:infinite, :, 0] = -float("inf")
    kw = dict(softcap=cap, slopes=sl / 64 if slopes else None)
    o, lse = tokens.attention(q, k, v, cq, ck, lq, lk, **kw)
    want, want_lse, mass = reference(q, k, v, cq, ck, d ** -0.5, **kw)
    e = 2.0 ** -18 * (1 + cap + (float(sl.max()) / 64 * lk if slopes else 0))
    assert ((lse.double() - want_lse).abs() <= e).all()
    assert ((o.double() - want).abs() <= U[dtype] * want.abs() + (U[dtype] + e) * mass + 1e-7).all()


@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_a_score_that_is_not_finite_shows_across_stretches(d, dtype):
    """Few rows over a long cache: the stretch with the key is joined with those without."""
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([2], [9000], 4, 2, d, dtype)
    q[:, :, 0] = 1
    for j in (0, 700, 4500, 8999):
        for bad in (float("nan"), float("inf")):
            x = k.clone()
            x[j, 0] = 0
            x[j, 0, 0] = bad
            o, lse = tokens.attention(q, x, v, cq, ck, 2, 9000)
            clean, clean_lse = tokens.attention(q, k, v, cq, ck, 2, 9000)
            assert torch.isnan(o[:, :2]).all() and not (torch.isfinite(lse[:2]) | torch.isneginf(lse[:2])).any(), (j, bad)
            assert torch.equal(o[:, 2:], clean[:, 2:]) and torch.equal(lse[2:], clean_lse[2:])
