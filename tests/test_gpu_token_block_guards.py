"""What a token block refuses instead of answering wrongly."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _block(width=128, heads=2, key_heads=1, **kw):
    from promptmoge_b200.token_block import TokenBlock
    torch.manual_seed(0)
    return TokenBlock(width, heads, key_heads, **kw).cuda()


def _frame(n=20):
    from promptmoge_b200.token_block import grid_angles
    cos, sin = grid_angles(16, 8, 32)
    return cos, sin, torch.arange(n, dtype=torch.int32, device="cuda")


def test_second_derivatives_are_refused():
    from promptmoge_b200.token_block import Packing
    block = _block()
    cos, sin, place = _frame()
    x = torch.randn(20, 128, device="cuda", requires_grad=True)
    y = block(x, Packing([20]), cos, sin, place)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.square().sum().backward()
