"""Positions are reported where they choose an angle, and only there."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (33, torch.float32)])        # by vectors; any size
@pytest.mark.parametrize("pairs", [0, 8])
def test_positions_without_rotation_are_not_looked_at(d, dtype, pairs):
    from promptmoge_b200 import tokens
    from promptmoge_b200._lib import PmgError
    q, k = torch.randn(5, 2, d, device="cuda").to(dtype), torch.randn(5, 1, d, device="cuda").to(dtype)
    cos, sin = torch.ones(4, pairs, device="cuda"), torch.zeros(4, pairs, device="cuda")
    place = torch.tensor([0, -1, 3, 0, 1], dtype=torch.int32, device="cuda")
    tokens.check()
    for call in (lambda: tokens.qk_norm_rope(q, k, None, None, cos, sin, place),
                 lambda: tokens.qk_norm_rope_grad(q, k, q, k, None, None, cos, sin, place)):
        call()
        if pairs:
            with pytest.raises(PmgError):
                tokens.check()
        tokens.check()
