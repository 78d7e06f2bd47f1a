"""A transformer block over the encoder tokens of several frames, run by the token operators.

The refiner reads one token feature map per frame (`RefinerEngine.set_frame`: [B, channels, h, w] fp16).  `TokenBlock`
is the layer that makes or adapts such tokens: every frame is a document of h * w tokens that attend to each other with
rotated positions; it trains (`torch.autograd`, through the operators' own gradients; a second derivative raises) and,
with `causal`, serves streams token by token over a cache (`step`, which also takes prompts).

    block = TokenBlock(1024, heads=16, key_heads=4).cuda()
    feature = mix_frames(block, encoder_feature)          # [B, 1024, 30, 40] fp16, as set_frame takes it
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import tokens


class Packing:
    """Documents of the given lengths, packed one after another: their offsets on the device and the longest."""

    def __init__(self, lengths, device="cuda"):
        self.lengths = [int(n) for n in lengths]
        if any(n < 0 for n in self.lengths):
            raise ValueError("lengths must not be negative")
        ends = torch.tensor([0] + self.lengths, dtype=torch.int64).cumsum(0)
        if int(ends[-1]) > 2 ** 31 - 1024:
            raise ValueError("too many tokens for 32-bit offsets")
        self.total = int(ends[-1])
        self.longest = max(self.lengths, default=0)
        self.offsets = ends.to(torch.int32).to(device)


def grid_angles(h: int, w: int, pairs: int, base: float = 100.0, device="cuda"):
    """cos, sin [h * w, pairs] fp32 of a token grid in row-major order: the first half of the pairs turns with the row,
    the rest with the column."""
    rows = pairs // 2
    at = torch.arange(h * w, device=device)
    parts = []
    for n, place in ((rows, at // w), (pairs - rows, at % w)):
        freq = base ** (-torch.arange(n, device=device, dtype=torch.float32) / max(n, 1))
        parts.append(place.float()[:, None] * freq)
    angle = torch.cat(parts, 1)
    return angle.cos().contiguous(), angle.sin().contiguous()


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, activation, residual):
        save = activation != "none"
        y = tokens.linear(x, w, b, activation=activation, residual=residual, save_pre=save)
        y, pre = y if save else (y, None)
        ctx.save_for_backward(x, w, pre)
        ctx.activation, ctx.has = activation, (b is not None, residual is not None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = tokens.linear_grad(dy.to(x.dtype).contiguous(), x, w, pre=pre, activation=ctx.activation,
                                        bias_grad=ctx.has[0] and need[2], input_grad=need[0], weight_grad=need[1])
        return dx, dw, db, None, dy if ctx.has[1] else None


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions):
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        return tokens.qk_norm_rope(q, k, qw, kw, cos, sin, positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        g = tokens.qk_norm_rope_grad(dq.contiguous(), dk.contiguous(), q, k, qw, kw, cos, sin, positions)
        return (*g, None, None, None)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, longest, options):
        o, lse = tokens.attention(q, k, v, offsets, offsets, longest, longest, **options)
        ctx.save_for_backward(q, k, v, o, lse, offsets)
        ctx.longest, ctx.options = longest, options
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, offsets = ctx.saved_tensors
        g = tokens.attention_grad(do.contiguous(), o, lse, q, k, v, offsets, offsets, ctx.longest, ctx.longest,
                                  **ctx.options)
        return (*g, None, None, None)


class TokenCache:
    """Keys and values of `streams` streams with room for `room` tokens each.

    `lengths` (int32, on the device) says how many each holds and may be set, to 0 for a new stream.  `TokenBlock.step`
    raises before it writes where a stream has no room left.  It knows the lengths from its own steps and reads them anew
    when they were set (a tensor made in inference mode that was put in their place: only then).  What a replayed graph adds
    it does not see: a token without room then stays within its stream, on the last row, and the status word tells
    (`tokens.check`)."""

    def __init__(self, block: "TokenBlock", streams: int, room: int, device="cuda"):
        shape = (streams * room, block.key_heads, block.head)
        self.k, self.v = (torch.empty(shape, dtype=block.dtype, device=device) for _ in range(2))
        self.streams, self.room = streams, room
        self.offsets = torch.arange(streams + 1, dtype=torch.int32, device=device) * room
        with torch.inference_mode(False):                  # so that it tells when it was set, in inference mode too
            self.lengths = torch.zeros(streams, dtype=torch.int32, device=device)
        self._held, self._mark = [0] * streams, self._version()

    def _version(self):
        return self.lengths, None if self.lengths.is_inference() else self.lengths._version

    def after(self, packing: Packing) -> list:
        """The streams' lengths with the packing's tokens; ValueError where they have no room for them."""
        known = self._mark is not None and self._mark[0] is self.lengths and self._mark[1] == self._version()[1]
        if not known and not torch.cuda.is_current_stream_capturing():
            self._held, self._mark = self.lengths.tolist(), self._version()
        lengths = [held + new for held, new in zip(self._held, packing.lengths)]
        for stream, n in enumerate(lengths):
            if n > self.room:
                raise ValueError(f"stream {stream} holds {self._held[stream]} of {self.room} tokens: "
                                 f"{packing.lengths[stream]} more do not fit")
        return lengths

    def rows(self, packing_offsets, total: int):
        """Cache rows of the next tokens of every stream, and their positions."""
        at = torch.arange(total, device=self.lengths.device, dtype=torch.int32)
        stream = torch.searchsorted(packing_offsets, at, right=True) - 1
        place = at - packing_offsets[stream] + self.lengths[stream]
        return stream * self.room + place.clamp(0, self.room - 1), place

    def grow(self, packing: Packing, lengths: list) -> None:
        """Counts the packing's tokens in; lengths: what after() gave."""
        self.lengths += packing.offsets.diff()
        self._held = lengths
        self._mark = None if torch.cuda.is_current_stream_capturing() else self._version()


class TokenBlock(nn.Module):
    """x + attention(norm(x)), then x + MLP(norm(x)), over packed tokens [T, width] kept in fp32.

    heads query heads share key_heads key heads; queries and keys are normalised and rotated; causal, softcap and
    slopes as in tokens.attention."""

    def __init__(self, width: int, heads: int, key_heads: int | None = None, hidden: int | None = None,
                 dtype=torch.bfloat16, causal: bool = False, softcap: float = 0.0, slopes=None):
        super().__init__()
        key_heads = heads if key_heads is None else key_heads
        if width % heads or heads % key_heads:
            raise ValueError("heads must divide the width, key_heads the heads")
        self.width, self.heads, self.key_heads, self.head, self.dtype = width, heads, key_heads, width // heads, dtype
        self.causal, self.softcap = causal, float(softcap)
        hidden = 4 * width if hidden is None else hidden
        self.norm1, self.norm2 = nn.LayerNorm(width, eps=1e-6), nn.LayerNorm(width, eps=1e-6)

        def weight(n, k):
            return nn.Parameter((torch.randn(n, k) * k ** -0.5).to(dtype)), nn.Parameter(torch.zeros(n, dtype=dtype))
        self.qkv_w, self.qkv_b = weight((heads + 2 * key_heads) * self.head, width)
        self.out_w, self.out_b = weight(width, width)
        self.up_w, self.up_b = weight(hidden, width)
        self.down_w, self.down_b = weight(width, hidden)
        self.q_norm, self.k_norm = nn.Parameter(torch.ones(self.head)), nn.Parameter(torch.ones(self.head))
        self.register_buffer("slopes", slopes)

    def _rows(self, x, packing: Packing):
        if x.shape != (packing.total, self.width):
            raise ValueError(f"x must be [{packing.total}, {self.width}] for this packing, got {tuple(x.shape)}")
        return x.contiguous()

    def _project(self, x):
        h = _Linear.apply(self.norm1(x).to(self.dtype), self.qkv_w, self.qkv_b, "none", None)
        a, b = self.heads * self.head, (self.heads + self.key_heads) * self.head
        return (h[:, :a].unflatten(1, (self.heads, self.head)), h[:, a:b].unflatten(1, (self.key_heads, self.head)),
                h[:, b:].unflatten(1, (self.key_heads, self.head)))

    def _finish(self, x, o):
        x = _Linear.apply(o.flatten(1), self.out_w, self.out_b, "none", x)
        h = _Linear.apply(self.norm2(x).to(self.dtype), self.up_w, self.up_b, "gelu", None)
        return _Linear.apply(h, self.down_w, self.down_b, "none", x)

    def _options(self, prefix=None):
        return dict(causal=self.causal, softcap=self.softcap, slopes=self.slopes, prefix=prefix)

    def forward(self, x, packing: Packing, cos, sin, positions, prefix=None):
        """x [T, width] fp32 -> the same; positions [T] int32 into the angle table; prefix [documents] int32."""
        x = self._rows(x, packing)
        q, k, v = self._project(x)
        q, k = _NormRope.apply(q, k, self.q_norm, self.k_norm, cos, sin, positions)
        return self._finish(x, _Attention.apply(q, k, v, packing.offsets, packing.longest, self._options(prefix)))

    @torch.no_grad()
    def step(self, x, packing: Packing, cache: TokenCache, cos, sin):
        """The next tokens of every stream (packing: how many of each; one at a time, or a prompt), their keys and
        values appended to the cache; ValueError where a stream has no room for them."""
        if not self.causal:
            raise ValueError("serving token by token needs a causal block")
        if len(packing.lengths) != cache.streams:
            raise ValueError(f"the cache holds {cache.streams} streams, got {len(packing.lengths)}")
        lengths = cache.after(packing)
        x = self._rows(x, packing)
        rows, place = cache.rows(packing.offsets, packing.total)
        q, k, v = self._project(x)
        q, k = tokens.qk_norm_rope(q, k, self.q_norm, self.k_norm, cos, sin, place)
        cache.k[rows], cache.v[rows] = k, v
        cache.grow(packing, lengths)
        o, _ = tokens.attention(q, cache.k, cache.v, packing.offsets, cache.offsets, packing.longest, cache.room,
                                k_len=cache.lengths, **self._options())
        return self._finish(x, o)


def mix_frames(block: TokenBlock, feature: torch.Tensor) -> torch.Tensor:
    """The block over a batch of encoder feature maps [B, width, h, w]: every frame's tokens attend within the frame.
    Returns fp16 [B, width, h, w], what RefinerEngine.set_frame and Refiner.refine take as encoder_feature."""
    B, C, h, w = feature.shape
    if C != block.width:
        raise ValueError(f"the block is {block.width} wide, the feature map {C}")
    x = feature.float().flatten(2).transpose(1, 2).reshape(B * h * w, C)
    cos, sin = grid_angles(h, w, block.head // 2, device=feature.device)
    place = torch.arange(h * w, dtype=torch.int32, device=feature.device).repeat(B)
    y = block(x, Packing([h * w] * B, feature.device), cos, sin, place)
    return y.view(B, h, w, C).permute(0, 3, 1, 2).to(torch.float16).contiguous()
