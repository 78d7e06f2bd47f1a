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
