"""The token operators' entry points without a GPU: refused arguments, workspace sizes, and no CPU path."""
import pytest
import torch

from promptmoge_b200 import _lib, tokens

BF16, F16, F32 = tokens.BF16, tokens.F16, tokens.F32
P = 1 << 12          # a pointer that is never followed: every call below is refused first


def test_linear_refusals():
    f = _lib.load().pmg_linear

    def call(x=P, ldx=64, w=P, ldw=64, dtype=BF16, M=40, N=64, K=64, act=0, y=P, ldy=64, ws=None, size=0):
        return f(x, ldx, w, ldw, dtype, M, N, K, None, act, None, 0, 0, y, ldy, None, 0, ws, size, None, None)
    assert call(M=0) == 0
    assert call(dtype=F32) == 5
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(act=4), dict(x=None), dict(w=None), dict(y=None), dict(ldx=63),
                dict(ldw=1), dict(ldy=8)):
        assert call(**bad) == 1, bad
    need = _lib.load().pmg_linear_workspace_bytes(40, 64, 65, 1, 1)
    assert need > 0 and call(K=65, ldx=65, ldw=65, ws=P, size=need - 1) == 1
    assert _lib.load().pmg_linear_workspace_bytes(32, 64, 65, 1, 1) == 0            # few rows need none


def test_linear_grad_refusals():
    f = _lib.load().pmg_linear_grad

    def call(dy=P, x=P, w=P, dtype=BF16, M=4, N=64, K=64, pre=None, act=0, dx=P, dw=None, db=None, size=0):
        return f(dy, 64, x, 64, w, 64, dtype, M, N, K, pre, 64, act, dx, 64, dw, 64, db, P, size, None, None)
    assert call(dtype=F32) == 5
    for bad in (dict(dy=None), dict(w=None), dict(act=3), dict(dx=None, dw=P, x=None), dict(M=-1), dict(db=P)):
        assert call(**bad) == 1, bad
    query = _lib.load().pmg_linear_grad_workspace_bytes
    assert query(100, 64, 64, 3, 0, 0, 0, 1) >= 100 * 64 * 2 + 64 * 4            # dz and the bias sums
    assert query(0, 64, 64, 3, 0, 0, 0, 1) == 0


def test_norm_rope_refusals():
    f = _lib.load().pmg_qk_norm_rope

    def call(q=P, k=P, dtype=BF16, T=3, Hq=2, Hk=1, D=64, rot=64, cos=P, sin=P, places=8, qo=P, ko=P):
        return f(q, 128, 64, k, 64, 64, dtype, T, Hq, Hk, D, rot, None, None, cos, sin, places, None, 1e-6, 0, qo, 128,
                 64, ko, 64, 64, None, None)
    assert call(T=0) == 0 and call(Hq=0, Hk=0) == 0
    assert call(dtype=7) == 5 and call(D=257) == 5
    for bad in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(cos=None), dict(sin=None), dict(rot=63),
                dict(rot=66), dict(rot=-2), dict(places=0), dict(T=-1), dict(D=0)):
        assert call(**bad) == 1, bad


def test_attention_refusals():
    f = _lib.load().pmg_attention

    def call(q=P, k=P, v=P, dtype=BF16, Tq=9, Tk=9, Hq=4, Hk=2, D=64, cu_q=P, cu_k=P, docs=1, max_q=9, max_k=9,
             scale=0.1, softcap=0.0, o=P, lse=P, tok=256):
        return f(q, tok, 64, k, 128, 64, v, 128, 64, dtype, Tq, Tk, Hq, Hk, D, cu_q, cu_k, None, docs, max_q, max_k,
                 scale, 0, None, softcap, None, o, 256, 64, lse, None, 0, None, None)
    assert call(Tq=0) == 0 and call(docs=0) == 0
    assert call(dtype=F32) == 5 and call(D=136) == 5 and call(D=60) == 5
    for bad in (dict(q=None), dict(o=None), dict(lse=None), dict(cu_q=None), dict(cu_k=None), dict(Hk=3), dict(Hk=0),
                dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0), dict(docs=-1), dict(max_q=-1), dict(tok=257),
                dict(q=P + 2)):
        assert call(**bad) == 1, bad
    query = _lib.load().pmg_attention_workspace_bytes
    assert query(1, 16, 4, 128, 4, 65501) > 0 and query(1, 16, 4, 128, 5, 65501) == 0 and query(64, 4, 4, 64, 1, 64) == 0


def test_attention_grad_refusals():
    f = _lib.load().pmg_attention_grad

    def call(dtype=BF16, Tq=9, Hq=4, Hk=2, D=64, lse=P, dq=P, size=1 << 30, scale=0.1):
        return f(P, 256, 64, P, 256, 64, lse, P, 256, 64, P, 128, 64, P, 128, 64, dtype, Tq, 9, Hq, Hk, D, P, P, None, 1,
                 scale, 0, None, 0.0, None, dq, 256, 64, P, 128, 64, P, 128, 64, P, size, None, None)
    assert call(dtype=F32) == 5
    for bad in (dict(lse=None), dict(dq=None), dict(dq=P + 8), dict(size=16), dict(scale=-1.0), dict(Hk=3)):
        assert call(**bad) == 1, bad


def test_no_cpu_path():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    q = torch.zeros(2, 1, 8, dtype=torch.bfloat16)
    cu = torch.tensor([0, 2], dtype=torch.int32)
    angles = torch.zeros(2, 4)
    for f in (lambda: tokens.linear(x, w), lambda: tokens.linear_grad(x, x, x), lambda: tokens.attention(q, q, q, cu, cu, 2, 2),
              lambda: tokens.qk_norm_rope(q, q, None, None, angles, angles)):
        with pytest.raises(ValueError, match="no CPU path"):
            f()
