"""What only the data shows is reported: offsets and lengths that leave their tensors, documents over max_q."""
import pytest
import torch

from attention_reference import offsets
from test_gpu_tokens_attention import make

pytestmark = pytest.mark.gpu


def words(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def reports(call):
    from promptmoge_b200 import tokens
    from promptmoge_b200._lib import PmgError
    tokens.check()
    call()
    with pytest.raises(PmgError):
        tokens.check()
    tokens.check()                                         # told once


BAD = [dict(cu_q=(0, 60, 101)), dict(cu_q=(-1, 60, 100)), dict(cu_k=(0, 70, 131)), dict(cu_k=(-5, 70, 130)), dict(cu_q=(0, 90, 60)),
       dict(cu_k=(0, 130, 70)), dict(k_len=(70, 61)), dict(k_len=(-1, 60)), dict(cu_q=(60, 60, 30))]


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_offsets_and_lengths_are_reported(bad, causal, d):
    """By the tile, and in the gradient."""
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([60, 40], [70, 60], 2, 1, d, torch.float16)
    args = dict(cu_q=cq, cu_k=ck, k_len=None) | {n: words(*x) for n, x in bad.items()}
    o, lse = torch.zeros_like(q), torch.zeros(2, 100, device="cuda")
    reports(lambda: tokens.attention(q, k, v, max_q=60, max_k=70, causal=causal, out=o, **args))
    reports(lambda: tokens.attention_grad(q, o, lse, q, k, v, max_q=60, max_k=70, causal=causal, **args))


@pytest.mark.parametrize("bad", BAD)
def test_offsets_and_lengths_are_reported_for_few_rows(bad):
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([60, 40], [70, 60], 1, 1, 64, torch.float16)
    args = dict(cu_q=cq, cu_k=ck, k_len=None) | {n: words(*x) for n, x in bad.items()}
    if "cu_q" not in bad:
        args["cu_q"] = words(0, 3, 6)
    reports(lambda: tokens.attention(q, k, v, max_q=3, max_k=70, **args))


@pytest.mark.parametrize("causal", [False, True])
def test_a_document_longer_than_max_q_is_reported_by_the_tile(causal):
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([20, 30, 25], [40, 40, 40], 2, 1, 64, torch.float16)
    tokens.attention(q, k, v, cq, ck, 30, 40, causal=causal)
    tokens.check()
    reports(lambda: tokens.attention(q, k, v, cq, ck, 29, 40, causal=causal))


@pytest.mark.parametrize("lk", [40, 9000])
def test_queries_although_max_q_is_zero(lk):
    from promptmoge_b200 import tokens
    q, k, v, cq, ck, _ = make([3], [lk], 2, 1, 64, torch.float16)
    reports(lambda: tokens.attention(q, k, v, cq, ck, 0, lk))
    none = words(0, 0)
    tokens.attention(q, k, v, none, ck, 0, lk)             # documents without queries: nothing to report
    tokens.check()


def test_any_upper_bound_of_the_keys():
    """max_k only chooses how the keys are shared out: the largest int32 serves every document."""
    from promptmoge_b200 import tokens
    for docs, hk in ((1, 1), (3, 2), (444, 8)):
        lk = [(37 * i) % 90 + 1 for i in range(docs)]
        q, k, v, cq, ck, _ = make([1] * docs, lk, hk, hk, 64, torch.float16)
        want = tokens.attention(q, k, v, cq, ck, 1, max(lk))
        got = tokens.attention(q, k, v, cq, ck, 1, 2 ** 31 - 1)
        tokens.check()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for most in (dict(max_k=2 ** 31), dict(max_q=2 ** 32 + 1, max_k=90)):
        with pytest.raises(ValueError):
            tokens.attention(q, k, v, cq, ck, **(dict(max_q=1) | most))
