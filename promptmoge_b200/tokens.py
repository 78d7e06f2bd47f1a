"""Token operators: the layers of a transformer block over packed tokens, as CUDA kernels of libpmg_b200.

  linear / linear_grad                  act(x W^T + b) + r in one pass, and the gradients of x, W, b
  qk_norm_rope / qk_norm_rope_grad      per-head norm of queries and keys with the position rotation, and its gradient
  attention / attention_grad            attention within documents: causal, prefix, capped scores, distance bias

Tokens of several frames (or streams) are packed one after another along the first axis.  Tensors are CUDA tensors of
one device, floating point, with contiguous innermost axis and otherwise any strides; kernels run on that device's
current stream, allocate outputs and scratch from torch's allocator and never synchronise.  Sums, norms and softmax
statistics are fp32.  What a kernel finds wrong with the data (a position outside the angle table, a wait that ran out)
is kept in a status word per device: `check()` reads it.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import PmgError, STATUS

F32, F16, BF16 = 0, 1, 2
_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}

_status_words: dict = {}
_fn: dict = {}


def _call(name, *args):
    f = _fn.get(name)
    if f is None:
        f = _fn[name] = getattr(_lib.load(), name)
    rc = f(*args)
    if rc != 0:
        raise PmgError(name, rc)


def _query(name, *args):
    f = _fn.get(name)
    if f is None:
        f = _fn[name] = getattr(_lib.load(), name)
    return f(*args)


def _status(index: int) -> int:
    word = _status_words.get(index)
    if word is None:
        word = _status_words[index] = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
        torch.cuda.current_stream(word.device).synchronize()    # zeroed before any other stream's kernel sees it
    return word.data_ptr()


def check(device=None) -> None:
    """Waits for the device, raises PmgError if a token operator on it has failed since the last check, and clears
    the status word."""
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    torch.cuda.synchronize(index)
    word = _status_words.get(index)
    code = 0 if word is None else int(word.item())
    if code:
        word.zero_()
        raise PmgError("token operator (" + STATUS.get(code, str(code)) + ")", code)


class _On:
    """Makes a tensor's device current where it is not."""
    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _dev(t, name, dim, index=None, dtypes=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (no CPU path)")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} axes, got shape {tuple(t.shape)}")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if index is not None and t.get_device() != index:
        raise ValueError(f"{name} is on another device")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous along its last axis")
    return t


_HALF = (torch.float16, torch.bfloat16)
_HALF_OR_F32 = (torch.float16, torch.bfloat16, torch.float32)


def _shape(t, shape, name):
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _ld(t):
    """Row stride; one that the row count leaves without meaning is taken as the row length."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _row(t):
    """(pointer, row stride) and whether the tensor-core path has to copy rows to 16-byte boundaries."""
    p, ld = t.data_ptr(), _ld(t)
    return p, ld, int(bool(p & 15 or ld & 7))


def _rows_ok(t, name):
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: rows must not overlap")
    return t


# ----------------------------------------------------------------------------------------------------------------- #
# Linear layers
# ----------------------------------------------------------------------------------------------------------------- #
def linear(x, w, bias=None, activation: str = "none", residual=None, save_pre: bool = False, out_dtype=None,
           out=None):
    """act(x w^T + bias) + residual.  x [M, K], w [N, K], bias [N] of one 16-bit type; residual [M, N] of the output's
    type; activation "none", "relu", "silu" or "gelu" (erf).  The output has x's type, or torch.float32 (out_dtype, or
    the residual's type where out_dtype is not given).  out: a tensor to write to (it may be the residual).  With
    save_pre, returns (y, x w^T + bias), the second for linear_grad."""
    _dev(x, "x", 2, None, _HALF)
    index = x.get_device()
    dt = x.dtype
    _dev(w, "w", 2, index, (dt,))
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"w must be [N, {K}], got {tuple(w.shape)}")
    if N < 1 or K < 1:
        raise ValueError("w must not be empty")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    _rows_ok(x, "x")
    _rows_ok(w, "w")
    if bias is not None:
        _shape(_dev(bias, "bias", 1, index, (dt,)), (N,), "bias")
    if residual is not None:
        _shape(_rows_ok(_dev(residual, "residual", 2, index, (dt, torch.float32)), "residual"), (M, N), "residual")
    odt = out_dtype if out_dtype is not None else (residual.dtype if residual is not None else dt)
    if odt != dt and odt != torch.float32:
        raise TypeError(f"out_dtype must be {dt} or torch.float32, got {odt}")
    if residual is not None and residual.dtype != odt:
        raise TypeError(f"residual must have the output's type {odt}, got {residual.dtype}")
    if out is None:
        y = torch.empty((M, N), dtype=odt, device=x.device)
    else:
        y = _rows_ok(_dev(out, "out", 2, index, (odt,)), "out")
        _shape(y, (M, N), "out")
    pre = torch.empty((M, N), dtype=dt, device=x.device) if save_pre else None
    if M:
        xp, ldx, px = _row(x)
        wp, ldw, pw = _row(w)
        need = _query("pmg_linear_workspace_bytes", M, N, K, px, pw)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        with _On(index) as stream:
            _call("pmg_linear", xp, ldx, wp, ldw, _DTYPES[dt], M, N, K, bias.data_ptr() if bias is not None else None,
                  act, residual.data_ptr() if residual is not None else None,
                  _ld(residual) if residual is not None else 0, int(odt == torch.float32), y.data_ptr(), _ld(y),
                  pre.data_ptr() if save_pre else None, N, ws.data_ptr() if need else None, need, _status(index),
                  stream)
    return (y, pre) if save_pre else y


def linear_grad(dy, x, w, pre=None, activation: str = "none", bias_grad: bool = True, input_grad: bool = True,
                weight_grad: bool = True):
    """Gradients (dx, dw, dbias) of linear() for dy [M, N], the gradient of its output, in x's type (dy too); None for
    one that is not asked for.  pre: the second output of linear(..., save_pre=True), needed unless the activation is
    "none".  The residual's gradient is dy itself."""
    _dev(x, "x", 2, None, _HALF)
    index, dt = x.get_device(), x.dtype
    _dev(w, "w", 2, index, (dt,))
    _dev(dy, "dy", 2, index, (dt,))
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K or N < 1 or K < 1:
        raise ValueError(f"w must be [N, {K}], got {tuple(w.shape)}")
    _shape(dy, (M, N), "dy")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if act and pre is None:
        raise ValueError("pre (linear(..., save_pre=True)) is needed for an activation's gradient")
    for t, name in ((x, "x"), (w, "w"), (dy, "dy")):
        _rows_ok(t, name)
    if act:
        _shape(_rows_ok(_dev(pre, "pre", 2, index, (dt,)), "pre"), (M, N), "pre")
    dx = torch.empty((M, K), dtype=dt, device=x.device) if input_grad else None
    dw = torch.empty((N, K), dtype=dt, device=x.device) if weight_grad else None
    db = torch.empty(N, dtype=dt, device=x.device) if bias_grad else None
    xp, ldx, px = _row(x)
    wp, ldw, pw = _row(w)
    yp, ldy, py = _row(dy)
    need = _query("pmg_linear_grad_workspace_bytes", M, N, K, act, py, px if weight_grad else 0,
                  pw if input_grad else 0, int(bias_grad))
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    with _On(index) as stream:
        _call("pmg_linear_grad", yp, ldy, xp, ldx, wp, ldw, _DTYPES[dt], M, N, K, pre.data_ptr() if act else None,
              _ld(pre) if act else 0, act, dx.data_ptr() if input_grad else None, K,
              dw.data_ptr() if weight_grad else None, K, db.data_ptr() if bias_grad else None,
              ws.data_ptr() if need else None, need, _status(index), stream)
    return dx, dw, db


# ----------------------------------------------------------------------------------------------------------------- #
# Norm of queries and keys with the position rotation
# ----------------------------------------------------------------------------------------------------------------- #
def _heads(t, name, index, dtypes):
    """(pointer, token stride, head stride) of [T, H, D]."""
    _dev(t, name, 3, index, dtypes)
    return t.data_ptr(), t.stride(0), t.stride(1)


def _angles(cos, sin, positions, T, D, index):
    _dev(cos, "cos", 2, index, (torch.float32,))
    _dev(sin, "sin", 2, index, (torch.float32,))
    places, half = cos.shape
    _shape(sin, cos.shape, "sin")
    if 2 * half > D:
        raise ValueError(f"cos and sin rotate {2 * half} values of heads of {D}")
    if not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("cos and sin must be contiguous")
    if positions is not None:
        _shape(_dev(positions, "positions", 1, index, (torch.int32,)), (T,), "positions")
    elif T > places and half:
        raise ValueError(f"{T} tokens without positions need as many rows of cos and sin, got {places}")
    if half and T and places == 0:
        raise ValueError("cos and sin must not be empty")
    return places, half


def _weight(w, name, D, index):
    if w is None:
        return None
    _shape(_dev(w, name, 1, index, (torch.float32,)), (D,), name)
    return w.data_ptr()


def _qk(q, k):
    _dev(q, "q", 3, None, _HALF_OR_F32)
    index, dt = q.get_device(), q.dtype
    _dev(k, "k", 3, index, (dt,))
    T, Hq, D = q.shape
    if k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"k must be [{T}, heads, {D}], got {tuple(k.shape)}")
    if D < 1 or D > 256:
        raise ValueError(f"heads hold 1 to 256 values, got {D}")
    return index, dt, T, Hq, k.shape[1], D


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6, interleaved: bool = False,
                 out=None):
    """Queries [T, Hq, D] and keys [T, Hk, D] (fp32, fp16 or bf16), each head divided by its root mean square and
    multiplied by the weight ([D] fp32 or None), then its first 2 * cos.shape[1] values rotated by the angles of the
    token's position: cos, sin [places, pairs] fp32; positions [T] int32 (None: 0, 1, 2, ...).  Pairs are (i, i +
    pairs), or (2i, 2i + 1) when interleaved.  out: a pair of tensors to write to, which may be q and k themselves or
    rows of a cache.  Returns (q, k)."""
    index, dt, T, Hq, Hk, D = _qk(q, k)
    places, half = _angles(cos, sin, positions, T, D, index)
    if out is None:
        qo, ko = (torch.empty(t.shape, dtype=dt, device=q.device) for t in (q, k))
    else:
        qo, ko = out
        _shape(_dev(qo, "out[0]", 3, index, (dt,)), q.shape, "out[0]")
        _shape(_dev(ko, "out[1]", 3, index, (dt,)), k.shape, "out[1]")
    with _On(index) as stream:
        _call("pmg_qk_norm_rope", q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
              _DTYPES[dt], T, Hq, Hk, D, 2 * half, _weight(q_weight, "q_weight", D, index),
              _weight(k_weight, "k_weight", D, index), cos.data_ptr(), sin.data_ptr(), places,
              positions.data_ptr() if positions is not None else None, eps, int(interleaved), qo.data_ptr(),
              qo.stride(0), qo.stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1), _status(index), stream)
    return qo, ko


def qk_norm_rope_grad(dq, dk, q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6,
                      interleaved: bool = False):
    """Gradients (q, k, q_weight, k_weight) of qk_norm_rope() for the gradients dq, dk of its outputs and its inputs
    q, k; the weights' in fp32, None where there is no weight."""
    index, dt, T, Hq, Hk, D = _qk(q, k)
    places, half = _angles(cos, sin, positions, T, D, index)
    _shape(_dev(dq, "dq", 3, index, (dt,)), q.shape, "dq")
    _shape(_dev(dk, "dk", 3, index, (dt,)), k.shape, "dk")
    gq, gk = (torch.empty(t.shape, dtype=dt, device=q.device) for t in (q, k))
    gqw = torch.empty(D, dtype=torch.float32, device=q.device) if q_weight is not None else None
    gkw = torch.empty(D, dtype=torch.float32, device=q.device) if k_weight is not None else None
    need = 0
    if q_weight is not None or k_weight is not None:
        need = _query("pmg_qk_norm_rope_grad_workspace_bytes", D)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    with _On(index) as stream:
        _call("pmg_qk_norm_rope_grad", *_heads(dq, "dq", index, (dt,)), *_heads(dk, "dk", index, (dt,)),
              *_heads(q, "q", index, (dt,)), *_heads(k, "k", index, (dt,)), _DTYPES[dt], T, Hq, Hk, D, 2 * half,
              _weight(q_weight, "q_weight", D, index), _weight(k_weight, "k_weight", D, index), cos.data_ptr(),
              sin.data_ptr(), places, positions.data_ptr() if positions is not None else None, eps, int(interleaved),
              gq.data_ptr(), gq.stride(0), gq.stride(1), gk.data_ptr(), gk.stride(0), gk.stride(1),
              gqw.data_ptr() if gqw is not None else None, gkw.data_ptr() if gkw is not None else None,
              ws.data_ptr() if need else None, need, _status(index), stream)
    return gq, gk, gqw, gkw


# ----------------------------------------------------------------------------------------------------------------- #
# Attention over packed documents
# ----------------------------------------------------------------------------------------------------------------- #
def _aligned_heads(t, name, shape, index, dt):
    """(pointer, token stride, head stride) of [T, H, D] on 16-byte boundaries."""
    _dev(t, name, 3, index, (dt,))
    if shape is not None:
        _shape(t, shape, name)
    T, H, D = t.shape
    p, st, sh = t.data_ptr(), t.stride(0), t.stride(1)
    if T <= 1:
        st = H * D if sh == D or H <= 1 else (st + 7) // 8 * 8
    if H <= 1:
        sh = D
    if p & 15 or st & 7 or sh & 7:
        raise ValueError(f"{name}: heads must start on 16-byte boundaries (strides in multiples of 8 values)")
    return p, st, sh


def _packing(cu_q, cu_k, k_len, prefix, slopes, Hq, index):
    docs = cu_q.shape[0] - 1
    for t, name, n in ((cu_q, "cu_q", docs + 1), (cu_k, "cu_k", docs + 1), (k_len, "k_len", docs),
                       (prefix, "prefix", docs)):
        if t is not None:
            _shape(_dev(t, name, 1, index, (torch.int32,)), (n,), name)
    if docs < 0:
        raise ValueError("cu_q must hold the documents' offsets, the total last")
    if slopes is not None:
        _shape(_dev(slopes, "slopes", 1, index, (torch.float32,)), (Hq,), "slopes")
    return docs


def _attention_shapes(q, k, v):
    _dev(q, "q", 3, None, _HALF)
    index, dt = q.get_device(), q.dtype
    Tq, Hq, D = q.shape
    _dev(k, "k", 3, index, (dt,))
    Tk, Hk, _ = k.shape
    if k.shape[2] != D or Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError(f"k must be [keys, heads, {D}] with a number of heads that divides {Hq}, got {tuple(k.shape)}")
    _shape(v, k.shape, "v")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"heads must hold a multiple of 8 values, 8 to 128, got {D}")
    return index, dt, Tq, Tk, Hq, Hk, D


def _score(scale, D, softcap, causal, prefix, max_q, max_k):
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf") or not 0.0 <= softcap < float("inf"):
        raise ValueError("scale must be positive and softcap not negative, both finite")
    if max_q < 0 or max_k < 0:
        raise ValueError("max_q and max_k must not be negative")
    if prefix is not None and not causal:
        raise ValueError("prefix needs causal (without it every key is seen)")
    return scale


def attention(q, k, v, cu_q, cu_k, max_q: int, max_k: int, scale: float | None = None, causal: bool = False,
              prefix=None, softcap: float = 0.0, slopes=None, k_len=None, out=None):
    """Attention within documents.  q [Tq, Hq, D], k and v [Tk, Hk, D] of one 16-bit type, Hq a multiple of Hk; cu_q,
    cu_k [documents + 1] int32: document d holds queries cu_q[d] .. cu_q[d+1] and keys cu_k[d] .. cu_k[d+1], or only
    the first k_len[d] of these (int32: a cache with spare room).  max_q, max_k: the most queries and keys of any
    document.  Query i stands at place p = i + Lk - Lq among its document's keys; causal: it sees keys j <= p, and j <
    prefix[d] (int32) where prefix is given.  Scores: scale (default D ** -0.5) times q.k, through softcap *
    tanh(. / softcap) if softcap is not 0, less slopes[h] (fp32) * |p - j| if slopes are given.

    Returns (o [Tq, Hq, D], lse [Hq, Tq] fp32).  Rows that see no key give 0 and -inf.  max_q * Hq / Hk <= 16 (token by
    token) takes the kernel that reads the keys once for all rows."""
    index, dt, Tq, Tk, Hq, Hk, D = _attention_shapes(q, k, v)
    docs = _packing(cu_q, cu_k, k_len, prefix, slopes, Hq, index)
    scale = _score(scale, D, softcap, causal, prefix, max_q, max_k)
    o = torch.empty((Tq, Hq, D), dtype=dt, device=q.device) if out is None else out
    lse = torch.empty((Hq, Tq), dtype=torch.float32, device=q.device)
    if not Tq:
        return o, lse
    oh = _aligned_heads(o, "out", (Tq, Hq, D), index, dt)
    need = _query("pmg_attention_workspace_bytes", docs, Hq, Hk, D, max_q, max_k)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    with _On(index) as stream:
        _call("pmg_attention", *_aligned_heads(q, "q", None, index, dt), *_aligned_heads(k, "k", None, index, dt),
              *_aligned_heads(v, "v", None, index, dt), _DTYPES[dt], Tq, Tk, Hq, Hk, D, cu_q.data_ptr(),
              cu_k.data_ptr(), k_len.data_ptr() if k_len is not None else None, docs, max_q, max_k, scale, int(causal),
              prefix.data_ptr() if prefix is not None else None, softcap,
              slopes.data_ptr() if slopes is not None else None, *oh, lse.data_ptr(),
              ws.data_ptr() if need else None, need, _status(index), stream)
    return o, lse


def attention_grad(do, o, lse, q, k, v, cu_q, cu_k, max_q: int, max_k: int, scale: float | None = None,
                   causal: bool = False, prefix=None, softcap: float = 0.0, slopes=None, k_len=None):
    """Gradients (dq, dk, dv) of attention() for do, the gradient of its output: o and lse are what it returned, the
    rest its arguments.  The slopes are constants of the score and get no gradient.  Key rows behind k_len get zeros."""
    index, dt, Tq, Tk, Hq, Hk, D = _attention_shapes(q, k, v)
    docs = _packing(cu_q, cu_k, k_len, prefix, slopes, Hq, index)
    scale = _score(scale, D, softcap, causal, prefix, max_q, max_k)
    _shape(_dev(lse, "lse", 2, index, (torch.float32,)), (Hq, Tq), "lse")
    if not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    doh = _aligned_heads(do, "do", q.shape, index, dt)
    oh = _aligned_heads(o, "o", q.shape, index, dt)
    dq, dk, dv = (torch.empty(t.shape, dtype=dt, device=q.device) for t in (q, k, v))
    need = _query("pmg_attention_grad_workspace_bytes", Tq, Hq)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    ks = (Hk * D, D)
    with _On(index) as stream:
        _call("pmg_attention_grad", *doh, *oh, lse.data_ptr(), *_aligned_heads(q, "q", None, index, dt),
              *_aligned_heads(k, "k", None, index, dt), *_aligned_heads(v, "v", None, index, dt), _DTYPES[dt], Tq, Tk,
              Hq, Hk, D, cu_q.data_ptr(), cu_k.data_ptr(), k_len.data_ptr() if k_len is not None else None, docs, scale,
              int(causal), prefix.data_ptr() if prefix is not None else None, softcap,
              slopes.data_ptr() if slopes is not None else None, dq.data_ptr(), Hq * D, D, dk.data_ptr(), *ks,
              dv.data_ptr(), *ks, ws.data_ptr(), need, _status(index), stream)
    return dq, dk, dv
