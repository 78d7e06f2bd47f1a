"""The token operators run together: a transformer block over packed frames against the same block in float64, its
gradients, serving token by token, and its output as the refiner's conditioning.

The block rounds every operand to 16 bits (u = 2^-8 in bf16) about ten times between input and output, each rounding's
effect on the result's norm at most a few u: results within 12 u of the float64 norm, gradients, which pass the block
twice, within 24 u."""
import pytest
import torch
import torch.nn.functional as F

from attention_reference import reference

pytestmark = pytest.mark.gpu


def _block(width=256, heads=4, key_heads=2, **kw):
    from promptmoge_b200.token_block import TokenBlock
    torch.manual_seed(0)
    return TokenBlock(width, heads, key_heads, **kw).cuda()


def _turn(x, w, cos, sin, place):
    n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    h = cos.shape[1]
    c, s = cos.double()[place][:, None], sin.double()[place][:, None]
    a, b = n[..., :h], n[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, n[..., 2 * h:]], -1)


def _exact(block, x, lengths, cos, sin, place, prefix=None):
    """The block's definition in float64 with autograd."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in block.named_parameters()}
    x = x.double().requires_grad_(True)
    h = F.layer_norm(x, (block.width,), p["norm1.weight"], p["norm1.bias"], 1e-6)
    h = h @ p["qkv_w"].t() + p["qkv_b"]
    a, b = block.heads * block.head, (block.heads + block.key_heads) * block.head
    q, k, v = h[:, :a].unflatten(1, (-1, block.head)), h[:, a:b].unflatten(1, (-1, block.head)), h[:, b:].unflatten(1, (-1, block.head))
    q, k = (_turn(t, p[n], cos, sin, place.long()) for t, n in ((q, "q_norm"), (k, "k_norm")))
    g, outs, at = block.heads // block.key_heads, [], 0
    for i, n in enumerate(lengths):
        qs, ks, vs = (t[at:at + n].transpose(0, 1) for t in (q, k, v))
        s = qs @ ks.repeat_interleave(g, 0).transpose(1, 2) * block.head ** -0.5
        if block.causal:
            j = torch.arange(n, device=x.device)
            s = s.masked_fill(~((j[None] <= j[:, None]) | (j[None] < (0 if prefix is None else int(prefix[i])))), float("-inf"))
        outs.append((s.softmax(-1) @ vs.repeat_interleave(g, 0)).transpose(0, 1))
        at += n
    x1 = x + torch.cat(outs).flatten(1) @ p["out_w"].t() + p["out_b"]
    h = F.gelu(F.layer_norm(x1, (block.width,), p["norm2.weight"], p["norm2.bias"], 1e-6) @ p["up_w"].t() + p["up_b"])
    return x1 + h @ p["down_w"].t() + p["down_b"], x, p


@pytest.mark.parametrize("causal", [False, True])
def test_block_and_gradients_equal_float64(causal):
    from promptmoge_b200 import tokens
    from promptmoge_b200.token_block import Packing, grid_angles
    block = _block(causal=causal)
    lengths = [130, 1, 200, 0, 37]
    cos, sin = grid_angles(20, 10, 32)
    place = torch.cat([torch.arange(n) for n in lengths]).to(torch.int32).cuda()
    x = torch.randn(sum(lengths), 256, device="cuda", requires_grad=True)
    prefix = torch.tensor([5, 1, 60, 0, 0], dtype=torch.int32, device="cuda") if causal else None
    y = block(x, Packing(lengths), cos, sin, place, prefix)
    c = torch.randn_like(y)
    y.backward(c)
    tokens.check()
    want, xd, p = _exact(block, x.detach(), lengths, cos, sin, place, prefix)
    want.backward(c.double())
    u = 2.0 ** -8
    assert (y.double() - want).norm() <= 12 * u * want.norm()
    assert (x.grad.double() - xd.grad).norm() <= 24 * u * xd.grad.norm()
    for n, t in block.named_parameters():
        assert (t.grad.double() - p[n].grad).norm() <= 24 * u * p[n].grad.norm(), n


def test_serving_equals_the_whole_sequence():
    """A prompt, then token by token over a cache with spare room, against the causal block over whole sequences."""
    from promptmoge_b200 import tokens
    from promptmoge_b200.token_block import Packing, TokenCache, grid_angles
    block = _block(causal=True)
    lengths, prompt = [45, 140, 33], [40, 135, 28]
    cos, sin = grid_angles(20, 10, 32)
    place = torch.cat([torch.arange(n) for n in lengths]).to(torch.int32).cuda()
    x = torch.randn(sum(lengths), 256, device="cuda")
    with torch.no_grad():
        whole = block(x, Packing(lengths), cos, sin, place).split(lengths)
    parts = x.split(lengths)
    cache = TokenCache(block, 3, 160)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    got = [[] for _ in lengths]
    for begin, count in [([0, 0, 0], prompt)] + [([n + i for n in prompt], [1, 1, 1]) for i in range(5)]:
        now = torch.cat([t[b:b + n] for t, b, n in zip(parts, begin, count)])
        y = block.step(now, Packing(count), cache, cos, sin)
        for g, t in zip(got, y.split(count)):
            g.append(t)
    tokens.check()
    for g, w in zip(got, whole):
        g = torch.cat(g)
        assert (g - w).norm() <= 12 * 2.0 ** -8 * w.norm()


def test_mixed_frames_condition_the_refiner():
    from promptmoge_b200 import synth
    from promptmoge_b200.refine import Refiner, synthetic_model
    from promptmoge_b200.token_block import mix_frames
    weights, clips = synthetic_model("B")
    sc = synth.make_scene(5, 48, 64, 8, synth.MODELS["B"]["model_channels"][-1])
    r = Refiner(weights, clips, model="B", height=48, width=64)
    block = _block(width=synth.ENC_CHANNELS, heads=16, key_heads=4, dtype=torch.float16)
    with torch.no_grad():
        feature = mix_frames(block, torch.from_numpy(sc.encoder_feature).cuda())
    assert feature.shape == sc.encoder_feature.shape and feature.dtype == torch.float16
    out, fit = r.refine(sc.point_coord, sc.lidar_depth, sc.lidar_conf, feature, sc.uv_bias)
    assert torch.isfinite(out).all() and fit[0]["ok"]
    plain, _ = r.refine(sc.point_coord, sc.lidar_depth, sc.lidar_conf, torch.from_numpy(sc.encoder_feature), sc.uv_bias)
    assert plain.shape == out.shape
    r.close()


def test_block_refusals():
    from promptmoge_b200.token_block import Packing, TokenBlock, TokenCache, grid_angles, mix_frames
    with pytest.raises(ValueError):
        TokenBlock(100, 3)
    with pytest.raises(ValueError):
        Packing([4, -1])
    block = _block()
    cos, sin = grid_angles(4, 4, 32)
    with pytest.raises(ValueError):
        block.step(torch.zeros(1, 256, device="cuda"), Packing([1]), TokenCache(block, 1, 8), cos, sin)
    with pytest.raises(ValueError):
        mix_frames(block, torch.zeros(1, 128, 4, 4, device="cuda"))


def test_reference_block_uses_the_same_attention():
    """The float64 block above and the attention tests' definition agree."""
    q, k, v = (torch.randn(9, 2, 16, device="cuda", dtype=torch.float64) for _ in range(3))
    cu = torch.tensor([0, 9], dtype=torch.int32)
    o = reference(q, k, v, cu, cu, 0.25)[0]
    s = (q.transpose(0, 1) @ k.transpose(0, 1).transpose(1, 2) * 0.25).softmax(-1)
    assert torch.allclose(o, (s @ v.transpose(0, 1)).transpose(0, 1))
