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


def test_a_full_cache_is_refused_before_it_is_written():
    from promptmoge_b200 import tokens
    from promptmoge_b200.token_block import Packing, TokenCache
    block = _block(causal=True)
    cos, sin, _ = _frame()
    cache = TokenCache(block, 3, 8)
    cache.k.zero_()
    cache.v.zero_()
    block.step(torch.randn(16, 128, device="cuda"), Packing([5, 3, 8]), cache, cos, sin)
    held = [t.clone() for t in (cache.k, cache.v, cache.lengths)]
    for more in ([4, 1, 0], [1, 1, 1], [0, 6, 0]):
        with pytest.raises(ValueError, match="do not fit"):
            block.step(torch.randn(sum(more), 128, device="cuda"), Packing(more), cache, cos, sin)
        assert all(torch.equal(a, b) for a, b in zip(held, (cache.k, cache.v, cache.lengths)))
    block.step(torch.randn(8, 128, device="cuda"), Packing([3, 5, 0]), cache, cos, sin)
    assert cache.lengths.tolist() == [8, 8, 8]
    assert torch.equal(cache.k[16:], held[0][16:]) and torch.equal(cache.k[:5], held[0][:5])
    cache.lengths[1] = 0                                   # a new stream in the second's place
    block.step(torch.randn(2, 128, device="cuda"), Packing([0, 2, 0]), cache, cos, sin)
    assert cache.lengths.tolist() == [8, 2, 8]
    with pytest.raises(ValueError, match="do not fit"):
        block.step(torch.randn(7, 128, device="cuda"), Packing([0, 7, 0]), cache, cos, sin)
    tokens.check()


def test_a_replayed_step_keeps_within_its_stream():
    """A captured step continues the streams as eager steps do; beyond the room it reports, and no neighbour is written."""
    from promptmoge_b200 import tokens
    from promptmoge_b200._lib import PmgError
    from promptmoge_b200.token_block import Packing, TokenCache
    block = _block(causal=True)
    cos, sin, _ = _frame()
    one, x = Packing([1, 0, 1]), torch.randn(2, 128, device="cuda")
    eager = TokenCache(block, 3, 8)
    want = [block.step(x, one, eager, cos, sin).clone() for _ in range(5)]
    cache = TokenCache(block, 3, 8)
    cache.k.zero_()
    cache.v.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block.step(x, one, cache, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.step(x, one, cache, cos, sin)
    for i in range(1, 5):
        graph.replay()
        assert torch.equal(y, want[i])
    assert cache.lengths.tolist() == [5, 0, 5]
    block.step(x, one, cache, cos, sin)                    # eager after replays: the lengths are read again
    tokens.check()
    for _ in range(4):
        graph.replay()
    with pytest.raises(PmgError):
        tokens.check()
    assert not cache.k[8:16].any() and not cache.v[8:16].any()
    with pytest.raises(ValueError, match="do not fit"):
        cache.lengths.clamp_(max=8)
        block.step(x, one, cache, cos, sin)


def test_tokens_and_packing_have_to_agree():
    """Tokens of no document have no result: they are refused, not left as memory came."""
    from promptmoge_b200.token_block import Packing, TokenCache
    block = _block(causal=True)
    cos, sin, place = _frame()
    x = torch.randn(20, 128, device="cuda")
    for lengths in ([19], [10, 11], [], [20, 1]):
        with pytest.raises(ValueError, match="for this packing"):
            block(x, Packing(lengths), cos, sin, place)
    with pytest.raises(ValueError, match="for this packing"):
        block.step(x, Packing([19]), TokenCache(block, 1, 32), cos, sin)
    with pytest.raises(ValueError, match="for this packing"):
        block(x[:, :64], Packing([20]), cos, sin, place)


def test_serving_in_inference_mode():
    from promptmoge_b200 import tokens
    from promptmoge_b200.token_block import Packing, TokenCache
    block = _block(causal=True)
    cos, sin, _ = _frame()
    x = torch.randn(4, 128, device="cuda")
    cache = TokenCache(block, 2, 4)
    want = block.step(x, Packing([3, 1]), cache, cos, sin)
    with torch.inference_mode():
        for made in (TokenCache(block, 2, 4), cache):
            made.lengths.zero_()
            assert torch.equal(block.step(x, Packing([3, 1]), made, cos, sin), want)
            with pytest.raises(ValueError, match="do not fit"):
                block.step(x[:2], Packing([2, 0]), made, cos, sin)
            made.lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
            assert torch.equal(block.step(x, Packing([3, 1]), made, cos, sin), want)
            with pytest.raises(ValueError, match="do not fit"):
                block.step(x[:2], Packing([2, 0]), made, cos, sin)
    tokens.check()
