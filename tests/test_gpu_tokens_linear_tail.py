"""Activations and their slopes relative to their own size, far into the negative tail.

The pre-activation is exact (the product is 0 and the bias is the value).  Tolerances, of the result: its rounding U,
and a quarter of it for the activation in 16 bits; in fp32 2^-19 for GELU (twice the fitted form's 1.2e-7, its
evaluation's 4e-7 and the exponential's 2.4e-7 together) and (|z| + 8) 2^-23 for SiLU, whose exponent is rounded to |z| 2^-24.
Below the smallest normal number the exponential is 0: z 2^-126 there, and fp16's own spacing."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# Phi by erfc: 1 + erf loses all of the tail behind -8.3, in float64 too
ACT = {"silu": torch.nn.functional.silu, "gelu": lambda z: z * 0.5 * torch.erfc(-z * 0.5 ** 0.5)}
TINY = {torch.bfloat16: 2.0 ** -118, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -118}


def points(dtype):
    z = torch.cat([torch.linspace(-13.5, 9, 901), torch.tensor([-300.0, -80.0, -60.0, -40.0, -17.0, -0.01, -1e-3, 0.0, 1e-3, 40.0])])
    return z.to(dtype).cuda()


@pytest.mark.parametrize("M,K", [(2, 24), (20, 24), (300, 24), (300, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out", ["own", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activation_relative_to_its_size(M, K, dtype, out, act):
    from promptmoge_b200 import tokens
    z = points(dtype)
    odt = torch.float32 if out == "fp32" else dtype
    x, w = torch.zeros(M, K, dtype=dtype, device="cuda"), torch.zeros(len(z), K, dtype=dtype, device="cuda")
    want = ACT[act](z.double())
    y = tokens.linear(x, w, z, activation=act, out_dtype=odt)
    assert y.dtype == odt
    fp32 = 2.0 ** -19 if act == "gelu" else (z.double().abs() + 8) * 2.0 ** -23
    share = U[odt] + fp32 if out == "fp32" else 1.25 * U[odt]
    err = (y.double() - want).abs() - (share * want.abs() + TINY[odt])
    worst = int(err.max(0)[0].argmax())
    assert (err <= 0).all(), (float(z[worst]), float(want[worst]), float(y[0, worst]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_slope_relative_to_its_size(dtype, act):
    """db of one row is the slope itself, rounded once; the slope is a sum of two terms, each as accurate as in fp32 above."""
    from promptmoge_b200 import tokens
    z = points(dtype)
    x, w = torch.zeros(1, 24, dtype=dtype, device="cuda"), torch.zeros(len(z), 24, dtype=dtype, device="cuda")
    db = tokens.linear_grad(torch.ones(1, len(z), dtype=dtype, device="cuda"), x, w, pre=z[None], activation=act)[2]
    zd = z.double().requires_grad_(True)
    want, = torch.autograd.grad(ACT[act](zd).sum(), zd)
    zd = zd.detach()
    if act == "gelu":
        size = 0.5 * torch.erfc(-zd * 0.5 ** 0.5) + zd.abs() * torch.exp(-zd * zd / 2) * 0.3989422804
        share = 2.0 ** -19 + zd * zd * 2.0 ** -24           # the exponent z^2 / 2 log2 e is rounded to 2^-24 of itself
    else:
        s = torch.sigmoid(zd)
        size = s + zd.abs() * s
        share = (zd.abs() + 8) * 2.0 ** -23
    assert ((db.double() - want).abs() <= U[dtype] * want.abs() + share * size + TINY[dtype]).all()
