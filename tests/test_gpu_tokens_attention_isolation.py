"""Rows do not depend, to the bit, on memory that is not theirs: what spare cache rows, rows of no document and other
documents hold, and what other rows see."""
import pytest
import torch

from attention_reference import offsets
from test_gpu_tokens_attention import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lq,lk,hq,hk", [(160, 160, 2, 1), (160, 500, 1, 1), (4, 200, 4, 1), (4, 3000, 4, 1)])      # by the tile; few rows
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_rows_do_not_follow_from_keys_that_others_see(lq, lk, hq, hk, d, dtype):
    """Keys that the causal mask hides from a row, but not from its neighbours: zero, or of the largest scores."""
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([lq], [lk], hq, hk, d, dtype)
    k *= torch.linspace(0.3, 3, lk, device="cuda")[:, None, None].to(dtype)
    first = lk - lq + (100 if lq > 100 else 2)             # hidden from the rows before place `first`
    got = []
    for fill in (0.0, 60.0):
        k[first:] = fill
        o, lse = tokens.attention(q, k, v, cq, ck, lq, lk, causal=True)
        got.append((o[:first - lk + lq], lse[:, :first - lk + lq]))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("lq", [[100, 3, 40], [4, 3, 2]])                 # by the tile; few rows
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_capped_scores_ignore_what_lies_outside(lq, d, dtype, slopes, causal):
    """Which form of tanh a row takes must not follow from keys behind a length, or from the neighbours' rows."""
    from promptmoge_b200 import tokens
    lk, room = [90, 40, 70], [110, 41, 200]
    q, k, v, cq, ck, sl = make(lq, lk, 4, 1, d, dtype, slopes=True, room=room)
    q *= 0.25                                              # scores well below half the cap
    do = torch.randn_like(q)
    used = torch.tensor(lk, dtype=torch.int32, device="cuda")
    kw = dict(causal=causal, softcap=20.0, slopes=sl if slopes else None, k_len=used)
    mine = slice(lq[0], lq[0] + lq[1])                     # the second document; the others change with the spare rows
    got = []
    for fill in (0.0, 200.0, float("nan")):
        for n, r, c in zip(lk, room, ck.tolist()):
            k[c + n:c + r] = fill
        if fill:
            q[:lq[0]] = 200.0
            q[lq[0] + lq[1]:] = -200.0
            k[room[0] + room[1]:] = fill
        o, lse = tokens.attention(q, k, v, cq, ck, max(lq), max(room), **kw)
        dq, dk, dv = tokens.attention_grad(do, o, lse, q, k, v, cq, ck, max(lq), max(room), **kw)
        keys = slice(room[0], room[0] + lk[1])
        got.append([t.clone() for t in (o[mine], lse[:, mine], dq[mine], dk[keys], dv[keys])])
    for other in got[1:]:
        for name, a, b in zip(("o", "lse", "dq", "dk", "dv"), got[0], other):
            assert torch.equal(a, b), name
    # keys that the causal mask hides from the first rows, huge against zero
    if causal:
        q, k, v, cq, ck, _ = make([160], [160], 2, 1, d, dtype)
        q *= 0.25
        firsts = []
        for fill in (0.0, 200.0):
            k[100:] = fill
            o, lse = tokens.attention(q, k, v, cq, ck, 160, 160, causal=True, softcap=20.0)
            firsts.append((o[:96], lse[:, :96]))
        assert all(torch.equal(a, b) for a, b in zip(*firsts))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(2, 2), (16, 1)])
def test_fp16_gradients_ignore_what_lies_outside(d, hq, hk):
    """Finite leftovers behind a cache's length, and rows behind the last document."""
    from promptmoge_b200 import tokens
    lq, lk, room = [200, 33, 0, 1], [700, 0, 30, 129], [720, 40, 64, 300]
    q, k, v, cq, ck, _ = make(lq + [16], lk, hq, hk, d, torch.float16, room=room)
    do = torch.randn_like(q) * 0.01
    cq, used = offsets(lq), torch.tensor(lk, dtype=torch.int32, device="cuda")
    got, own = [], sum(lq)
    for fill in (0.0, 6e4, -6e4):
        for n, r, c in zip(lk, room, ck.tolist()):
            k[c + n:c + r] = fill
            v[c + n:c + r] = fill
        for t in (q, do):
            t[own:] = fill
        out = torch.full_like(q, fill)
        o, lse = tokens.attention(q, k, v, cq, ck, 200, 720, causal=True, k_len=used, out=out)
        lse[:, own:] = 0
        dq, dk, dv = tokens.attention_grad(do, o, lse, q, k, v, cq, ck, 200, 720, causal=True, k_len=used)
        got.append([o[:own], lse[:, :own], dq[:own], dk, dv])
    tokens.check()
    for other in got[1:]:
        for name, a, b in zip(("o", "lse", "dq", "dk", "dv"), got[0], other):
            assert torch.equal(a, b), name


@pytest.mark.parametrize("d,hq,hk", [(64, 2, 1), (128, 4, 4)])
def test_fp16_gradients_of_a_document_are_its_own(d, hq, hk):
    """Large gradients and values in one document leave the bits of the others'."""
    from promptmoge_b200 import tokens
    lens = [130, 5, 300, 77]
    q, k, v, cq, ck, _ = make(lens, lens, hq, hk, d, torch.float16)
    do = torch.randn_like(q) * 2.0 ** -8
    keep = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    keep[135:435] = False

    def grads():
        o, lse = tokens.attention(q, k, v, cq, ck, 300, 300)
        return tokens.attention_grad(do, o, lse, q, k, v, cq, ck, 300, 300)
    want = grads()
    do[135:435] *= 2.0 ** 16
    v[135:435] *= 2.0 ** 10
    for a, b in zip(grads(), want):
        assert torch.equal(a[keep], b[keep])
