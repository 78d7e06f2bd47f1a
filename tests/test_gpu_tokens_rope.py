"""Per-head norm of queries and keys with the position rotation, and its gradient, against float64.

Tolerances: fp32 arithmetic on at most 256 terms keeps a value within 1e-6 of the row's scale; one rounding to the
output type adds its unit roundoff u.  The weights' gradients are fp32 sums of T * heads terms in short strands: within
1e-6 times the sum of the terms' sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}


def _exact(x, w, cos, sin, pos, eps, interleaved):
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    n = n if w is None else n * w
    h = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = (n[..., 0:2 * h:2], n[..., 1:2 * h:2]) if interleaved else (n[..., :h], n[..., h:2 * h])
    ra, rb = a * c - b * s, b * c + a * s
    turned = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([turned, n[..., 2 * h:]], -1)


def _case(T, Hq, Hk, D, rot, dtype, weight, seed=0, places=50):
    gen = torch.Generator(device="cuda").manual_seed(seed + T + D)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    fused = rand(T, (Hq + 2 * Hk) * D).to(dtype)
    q = fused[:, :Hq * D].unflatten(1, (Hq, D))
    k = fused[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
    ang = rand(places, rot // 2) * 3
    pos = torch.randint(0, places, (T,), generator=gen, device="cuda", dtype=torch.int32)
    qw, kw = (1 + 0.3 * rand(D), 1 + 0.3 * rand(D)) if weight else (None, None)
    return q, k, qw, kw, ang.cos(), ang.sin(), pos


CASES = [(1, 1, 1, 8, 8), (1, 16, 4, 64, 64), (3, 2, 1, 80, 40), (7, 5, 3, 36, 12), (5, 3, 1, 33, 6), (2, 1, 2, 1, 0),
         (64, 8, 8, 128, 96), (33, 4, 2, 256, 256), (300, 16, 4, 64, 32), (129, 6, 2, 200, 100), (4000, 16, 4, 32, 32),
         (2500, 20, 5, 128, 128)]


@pytest.mark.parametrize("T,Hq,Hk,D,rot", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weight", [False, True])
def test_forward_and_gradient(T, Hq, Hk, D, rot, dtype, interleaved, weight):
    from promptmoge_b200 import tokens
    q, k, qw, kw, cos, sin, pos = _case(T, Hq, Hk, D, rot, dtype, weight)
    out = tokens.qk_norm_rope(q, k, qw, kw, cos, sin, pos, eps=1e-5, interleaved=interleaved)
    gen = torch.Generator(device="cuda").manual_seed(5)
    dy = [torch.randn(t.shape, generator=gen, device="cuda").to(dtype) for t in (q, k)]
    got = tokens.qk_norm_rope_grad(*dy, q, k, qw, kw, cos, sin, pos, eps=1e-5, interleaved=interleaved)
    tokens.check()
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        xd = x.double().requires_grad_(True)
        wd = None if w is None else w.double().requires_grad_(True)
        y = _exact(xd, wd, cos, sin, pos.long(), 1e-5, interleaved)
        grads = torch.autograd.grad(y, [xd] if w is None else [xd, wd], dy[i].double())
        size = y.abs().amax(-1, keepdim=True)
        assert ((out[i].double() - y).abs() <= U[dtype] * y.abs() + 2e-6 * size + 1e-7).all()
        r = 1 / (xd.square().mean(-1, keepdim=True) + 1e-5).sqrt()
        size = r * dy[i].double().abs().amax(-1, keepdim=True) * (1 if w is None else w.abs().max()) * 4
        size = size * (1 + (xd.abs() * r).amax(-1, keepdim=True) * D ** 0.5)
        assert ((got[i].double() - grads[0]).abs() <= U[dtype] * grads[0].abs() + 2e-6 * size).all()
        if w is None:
            assert got[2 + i] is None
        else:
            n = (xd * r).detach().abs()
            terms = 2 * (n * dy[i].double().abs().amax(-1, keepdim=True)).sum((0, 1))
            assert ((got[2 + i].double() - grads[1]).abs() <= 2e-6 * terms + 1e-6).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(interleaved):
    from promptmoge_b200 import tokens
    q, k, qw, kw, cos, sin, pos = _case(6, 3, 2, 24, 16, torch.float32, True)
    c = [torch.randn_like(t) for t in (q, k)]
    g = tokens.qk_norm_rope_grad(*c, q, k, qw, kw, cos, sin, pos, interleaved=interleaved)

    def loss(a):
        return sum((_exact(a[i], a[2 + i], cos, sin, pos.long(), 1e-6, interleaved) * c[i].double()).sum() for i in (0, 1))
    base = [t.double() for t in (q, k, qw, kw)]
    for i in range(4):
        d = g[i].double()
        h = 1e-5 / d.norm()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        assert abs((loss(up) - loss(down)) / (2 * h) / d.square().sum() - 1) < 1e-5   # h^2 and fp32 terms


def test_in_place_and_into_a_cache():
    from promptmoge_b200 import tokens
    q, k, qw, kw, cos, sin, pos = _case(40, 4, 2, 64, 64, torch.bfloat16, True)
    want = tokens.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    cache = torch.zeros(100, 2, 64, dtype=torch.bfloat16, device="cuda")
    q2, _ = tokens.qk_norm_rope(q, k, qw, kw, cos, sin, pos, out=(q, cache[30:70]))
    assert q2.data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(cache[30:70], want[1])
    assert not cache[:30].any() and not cache[70:].any()


def test_positions_by_order_and_zero_rows():
    from promptmoge_b200 import tokens
    q, k, qw, kw, cos, sin, _ = _case(30, 4, 2, 64, 64, torch.bfloat16, True)
    q = q.clone()
    q[3] = 0
    a = tokens.qk_norm_rope(q, k, qw, kw, cos, sin)
    b = tokens.qk_norm_rope(q, k, qw, kw, cos, sin, torch.arange(30, device="cuda", dtype=torch.int32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not a[0][3].any()
    e = tokens.qk_norm_rope(q[:0], k[:0], qw, kw, cos, sin)
    assert e[0].shape == (0, 4, 64)
    g = tokens.qk_norm_rope_grad(q[:0], k[:0], q[:0], k[:0], qw, kw, cos, sin)
    assert not g[2].any() and not g[3].any()


def test_a_position_outside_the_table_is_reported():
    from promptmoge_b200 import tokens
    from promptmoge_b200._lib import PmgError
    q, k, qw, kw, cos, sin, pos = _case(10, 2, 1, 32, 32, torch.bfloat16, True)
    pos[4] = 50
    pos[5] = -1
    out = tokens.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    with pytest.raises(PmgError):
        tokens.check()
    tokens.check()
    pos[4] = pos[5] = 0
    assert torch.equal(out[0], tokens.qk_norm_rope(q, k, qw, kw, cos, sin, pos)[0])


def test_refusals():
    from promptmoge_b200 import tokens
    q, k, qw, kw, cos, sin, pos = _case(10, 2, 1, 32, 32, torch.bfloat16, True)
    bad = [dict(q=q.cpu()), dict(k=k[:5]), dict(k=k[..., :16]), dict(qw=qw[:5]), dict(cos=cos[:3]), dict(pos=pos[:3]),
           dict(cos=cos.repeat(1, 2), sin=sin.repeat(1, 2)), dict(q=q.transpose(1, 2))]
    for change in bad:
        a = dict(q=q, k=k, qw=qw, kw=kw, cos=cos, sin=sin, pos=pos) | change
        with pytest.raises(ValueError):
            tokens.qk_norm_rope(*a.values())
    for change in (dict(k=k.half()), dict(qw=qw.half()), dict(pos=pos.long())):
        a = dict(q=q, k=k, qw=qw, kw=kw, cos=cos, sin=sin, pos=pos) | change
        with pytest.raises(TypeError):
            tokens.qk_norm_rope(*a.values())
    with pytest.raises(ValueError):
        tokens.qk_norm_rope(q.repeat(10, 1, 1), k.repeat(10, 1, 1), qw, kw, cos, sin)
