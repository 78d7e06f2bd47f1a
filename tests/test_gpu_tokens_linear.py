"""Linear layers with a fused epilogue, and their gradients, against float64.

Tolerances.  u is the output type's unit roundoff (2^-8 bf16, 2^-11 fp16).  The
product's fp32 sums are bounded by (K/8 + 8) 2^-23 times the sum of |x w| (tensor cores may truncate once per step of at
most 16 terms); the activation's own error is at most 1.5e-5 plus its largest slope (1.13) times that.  Gradients add
one rounding of dz to the operands' type, at most u of each term."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}
ACT = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}


def _rand(gen, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _inputs(M, N, K, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + M + 7 * N + 13 * K)
    return (_rand(gen, M, K, dtype=dtype), _rand(gen, N, K, dtype=dtype, scale=K ** -0.5),
            _rand(gen, N, dtype=dtype), _rand(gen, M, N, dtype=dtype))


def _slack(x, w, K):
    return (K / 8 + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t())


SHAPES = [(1, 16, 8), (1, 4096, 1024), (7, 33, 29), (8, 1, 1), (9, 100, 257), (16, 64, 64), (31, 1026, 130),
          (33, 64, 64), (64, 17, 1026), (127, 129, 72), (129, 255, 1000), (200, 384, 64), (300, 1024, 520),
          (1200, 1024, 1026), (1000, 4096, 136), (4097, 260, 96), (2400, 1536, 1024)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_linear_equals_float64(M, N, K, dtype, act):
    from promptmoge_b200 import tokens
    x, w, b, r = _inputs(M, N, K, dtype)
    y, pre = tokens.linear(x, w, b, activation=act, residual=r, save_pre=True)
    tokens.check()
    z = x.double() @ w.double().t() + b.double()
    want = ACT[act](z) + r.double()
    slack = _slack(x, w, K) + 2.0 ** -22 * z.abs()
    assert ((pre.double() - z).abs() <= U[dtype] * z.abs() + slack + 1e-7).all()
    tol = U[dtype] * want.abs() + 1.13 * slack + 2.0 ** -22 * (want.abs() + r.double().abs()) + 1.5e-5
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (5, 1024, 1024), (130, 200, 264), (1200, 1024, 1026)])
@pytest.mark.parametrize("bias,resid", [(False, False), (True, True)])
def test_linear_float32_stream(M, N, K, bias, resid):
    """fp32 output and residual, updated in place."""
    from promptmoge_b200 import tokens
    x, w, b, r = _inputs(M, N, K, torch.bfloat16)
    r = r.float()
    want = x.double() @ w.double().t() + (b.double() if bias else 0) + (r.double() if resid else 0)
    y = tokens.linear(x, w, b if bias else None, residual=r if resid else None, out_dtype=torch.float32,
                      out=r if resid else None)
    assert y.dtype == torch.float32 and (not resid or y.data_ptr() == r.data_ptr())
    tol = _slack(x, w, K) + 2.0 ** -22 * want.abs() + 1e-6
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("M", [3, 20, 257])
def test_linear_strided_rows_and_odd_places(M):
    """Rows with a stride of their own, starting at odd places, and an output inside a larger tensor."""
    from promptmoge_b200 import tokens
    gen = torch.Generator(device="cuda").manual_seed(M)
    for off, ld in ((0, 136), (8, 160), (3, 133)):
        buf = _rand(gen, M, ld, dtype=torch.float16)
        x = buf[:, off:off + 96]
        wb = _rand(gen, 70, ld, dtype=torch.float16, scale=0.1)
        w = wb[:, off:off + 96]
        big = torch.full((M, 200), 7.0, dtype=torch.float16, device="cuda")
        tokens.linear(x, w, activation="silu", out=big[:, off:off + 70])
        z = x.double() @ w.double().t()
        want = ACT["silu"](z)
        tol = U[torch.float16] * want.abs() + 1.13 * _slack(x, w, 96) + 1.5e-5
        assert ((big[:, off:off + 70].double() - want).abs() <= tol).all()
        rest = torch.ones(200, dtype=torch.bool)
        rest[off:off + 70] = False
        assert (big[:, rest] == 7).all()


@pytest.mark.parametrize("M", [1, 200])
def test_linear_keeps_what_is_not_finite_in_its_row(M):
    from promptmoge_b200 import tokens
    x, w, b, _ = _inputs(M + 2, 300, 128, torch.bfloat16)
    x[1, 5] = float("nan")
    x[2, 5] = float("inf")
    for act in ACT:
        y = tokens.linear(x, w, b, activation=act)
        assert torch.isnan(y[1]).all()
        assert torch.isfinite(y[0]).all() and torch.isfinite(y[3:]).all()
    assert torch.isinf(tokens.linear(x, w, b)[2]).all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_activation_over_its_range(act):
    """x W^T with one-hot weights leaves x itself in front of the activation: the whole range, ends included."""
    from promptmoge_b200 import tokens
    v = torch.cat([torch.linspace(-12, 12, 8190), torch.tensor([-60000.0, 60000.0])]).cuda().to(torch.float16)
    x = torch.zeros(8192, 64, dtype=torch.float16, device="cuda")
    x[:, 0] = v
    w = torch.zeros(64, 64, dtype=torch.float16, device="cuda")
    w[:, 0] = 1
    for rows in (slice(0, 8192), slice(0, 8), slice(8184, 8192)):
        y = tokens.linear(x[rows], w, activation=act)[:, 0].double()
        want = ACT[act](v[rows].double())
        assert ((y - want).abs() <= U[torch.float16] * want.abs() + 1.5e-5).all()


GRADS = [(1, 16, 8), (1, 100, 64), (8, 33, 29), (33, 64, 72), (130, 257, 130), (1200, 1024, 1026), (999, 512, 264),
         (5000, 64, 96), (640, 4096, 1024)]


@pytest.mark.parametrize("M,N,K", GRADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_linear_grad_equals_float64(M, N, K, dtype, act):
    from promptmoge_b200 import tokens
    x, w, b, dy = _inputs(M, N, K, dtype, seed=1)
    pre = (x.double() @ w.double().t() + b.double()).to(dtype)
    dx, dw, db = tokens.linear_grad(dy, x, w, pre=pre, activation=act)
    tokens.check()
    z = pre.double().requires_grad_(True)
    dz, = torch.autograd.grad(ACT[act](z), z, dy.double())
    u, uz = U[dtype], 0.0 if act == "none" else U[dtype]

    def close(got, a, c, terms):
        want, size = a @ c, a.abs() @ c.abs()
        assert ((got.double() - want).abs() <= u * want.abs() + (uz + 2.0 ** -20 + (terms / 8 + 8) * 2.0 ** -23) * size
                + 1e-7).all()
    close(dx, dz, w.double(), N)
    close(dw, dz.t(), x.double(), M)
    want = dz.sum(0)
    assert ((db.double() - want).abs() <= u * want.abs() + (2.0 ** -20 + M * 2.0 ** -24) * dz.abs().sum(0) + 1e-7).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_linear_grad_against_differences(act):
    """The directional derivative of a float64 loss along the computed gradients, by central differences."""
    from promptmoge_b200 import tokens
    x, w, b, c = _inputs(96, 80, 64, torch.bfloat16, seed=2)
    _, pre = tokens.linear(x, w, b, activation=act, save_pre=True)
    dx, dw, db = (t.double() for t in tokens.linear_grad(c, x, w, pre=pre, activation=act))
    xd, wd, bd, cd = x.double(), w.double(), b.double(), c.double()

    def loss(xx, ww, bb):
        return (ACT[act](xx @ ww.t() + bb) * cd).sum()
    for i, g in enumerate((dx, dw, db)):
        h = 1e-4 / g.norm()
        up, down = [xd, wd, bd], [xd, wd, bd]
        up[i], down[i] = up[i] + h * g, down[i] - h * g
        slope = (loss(*up) - loss(*down)) / (2 * h)
        # the gradient's own rounding (bf16, dz and output) along itself: far below 1 %
        assert abs(slope / g.square().sum() - 1) < 1e-2


def test_linear_grad_parts_and_repeats():
    from promptmoge_b200 import tokens
    x, w, b, dy = _inputs(700, 320, 200, torch.bfloat16)
    pre = tokens.linear(x, w, b, save_pre=True)[1]
    every = tokens.linear_grad(dy, x, w, pre=pre, activation="gelu")
    again = tokens.linear_grad(dy, x, w, pre=pre, activation="gelu")
    assert all(torch.equal(a, c) for a, c in zip(every, again))
    for ask in range(8):
        part = tokens.linear_grad(dy, x, w, pre=pre, activation="gelu", input_grad=bool(ask & 1),
                                  weight_grad=bool(ask & 2), bias_grad=bool(ask & 4))
        for i in range(3):
            assert (part[i] is None) if not ask >> i & 1 else torch.equal(part[i], every[i])


def test_linear_without_rows():
    from promptmoge_b200 import tokens
    x, w, b, dy = _inputs(0, 24, 40, torch.bfloat16)
    assert tokens.linear(x, w, b, activation="gelu").shape == (0, 24)
    dx, dw, db = tokens.linear_grad(dy, x, w)
    assert dx.shape == (0, 40) and not dw.any() and not db.any()


def test_linear_on_another_stream():
    from promptmoge_b200 import tokens
    x, w, b, r = _inputs(400, 256, 256, torch.float16)
    want = tokens.linear(x, w, b, residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tokens.linear(x, w, b, residual=r)
    s.synchronize()
    assert torch.equal(got, want)


def test_linear_refusals():
    from promptmoge_b200 import tokens
    x, w, b, r = _inputs(4, 8, 16, torch.bfloat16)
    with pytest.raises(ValueError):
        tokens.linear(x.cpu(), w)
    with pytest.raises(TypeError):
        tokens.linear(x.float(), w.float())
    with pytest.raises(TypeError):
        tokens.linear(x, w.half())
    with pytest.raises(ValueError):
        tokens.linear(x, w[:, :8])
    with pytest.raises(ValueError):
        tokens.linear(x, w, activation="tanh")
    with pytest.raises(ValueError):
        tokens.linear(x, w, bias=b[:4])
    with pytest.raises(ValueError):
        tokens.linear(x, w, residual=r[:, :4])
    with pytest.raises(TypeError):
        tokens.linear(x, w, residual=r, out_dtype=torch.float32)
    with pytest.raises(ValueError):
        tokens.linear(x.t(), w)
    with pytest.raises(ValueError):
        tokens.linear(x[:1].expand(4, 16), w)
    with pytest.raises(ValueError):
        tokens.linear_grad(r, x, w, activation="gelu")


@pytest.mark.parametrize("M", [2, 20, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_activation_over_its_whole_range(M, dtype, act):
    """Pre-activations from far below to far above 0 (the bias alone, the product being 0), with +inf and NaN."""
    from promptmoge_b200 import tokens
    z = torch.cat([torch.linspace(-9, 9, 301), torch.tensor([-6e4, -300.0, -40.0, -17.0, -16.0, -15.9, 16.0, 300.0, 6e4])])
    z = z.to(dtype).cuda()
    x, w = torch.zeros(M, 24, dtype=dtype, device="cuda"), torch.zeros(len(z), 24, dtype=dtype, device="cuda")
    want = ACT[act](z.double())
    y = tokens.linear(x, w, z, activation=act)
    assert ((y.double() - want).abs() <= U[dtype] * want.abs() + 2.0 ** -22 * want.abs() + 1.5e-5).all()
    z = torch.tensor([float("inf"), float("nan"), 1.0] * 20, dtype=dtype, device="cuda")
    y = tokens.linear(x, torch.zeros(60, 24, dtype=dtype, device="cuda"), z, activation=act)
    assert (y[:, 0::3] == float("inf")).all() and torch.isnan(y[:, 1::3]).all() and torch.isfinite(y[:, 2::3]).all()


@pytest.mark.parametrize("M,N,K", [(40, 48, 64), (200, 130, 96), (2400, 1536, 1024)])
@pytest.mark.parametrize("off,ld", [(0, 1600), (16, 1616), (8, 1608), (1, 1601)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_output_and_residual_rows_on_any_boundary(M, N, K, off, ld, out):
    """Rows of 32-byte, 16-byte and element alignment, residual and output in one larger tensor, nothing else touched."""
    from promptmoge_b200 import tokens
    x, w, b, r = _inputs(M, N, K, torch.bfloat16)
    big = torch.full((M, ld), 5.0, dtype=out, device="cuda")
    place = big[:, off:off + N]
    place.copy_(r)
    want = x.double() @ w.double().t() + b.double() + r.double()
    tokens.linear(x, w, b, residual=place, out=place)
    tol = U[out] * want.abs() + _slack(x, w, K) + 2.0 ** -22 * (want.abs() + r.double().abs()) + 1e-6
    assert ((place.double() - want).abs() <= tol).all()
    assert (big[:, :off] == 5).all() and (big[:, off + N:] == 5).all()
