"""Token operators: the layers of a transformer block over packed tokens, as CUDA kernels of libpmg_b200.

  linear / linear_grad                  act(x W^T + b) + r in one pass, and the gradients of x, W, b
  qk_norm_rope / qk_norm_rope_grad      per-head norm of queries and keys with the position rotation, and its gradient
  attention / attention_grad            attention within documents: causal, prefix, capped scores, distance bias

Tokens of several frames (or streams) are packed one after another along the first axis.  Tensors are CUDA tensors of
one device, floating point, with contiguous innermost axis and otherwise any strides; kernels run on that device's
current stream, allocate outputs and scratch from torch's allocator and never synchronise.  Sums, norms and softmax
statistics are fp32.  What a kernel finds wrong with the data (a position outside the angle table, a document longer than
max_q, a wait that ran out) is kept in a status word per device: `check()` reads it.

Results carry no autograd graph, whatever their inputs require: the *_grad functions are the backward passes, and
`token_block.TokenBlock` puts both into one.
"""
from __future__ import annotations

import functools
import threading

import torch

from . import _lib
from ._lib import PmgError, STATUS

F32, F16, BF16 = 0, 1, 2
_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}

_status_words: dict = {}
_status_ptrs: dict = {}
_status_lock = threading.Lock()
_fn: dict = {}
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream


# Small calls are bound by the host: a call's checks read each attribute of a tensor once, and only a call that fails
# them runs the functions that say why.
def _call(name, *args):
    f = _fn.get(name)
    if f is None:
        f = _fn[name] = getattr(_lib.load(), name)
    rc = f(*args)
    if rc:
        raise PmgError(name, rc)


@functools.lru_cache(maxsize=4096)
def _query(name, *sizes):
    """A workspace size, which depends on a call's sizes alone."""
    return getattr(_lib.load(), name)(*sizes)


def _status(index: int) -> int:
    ptr = _status_ptrs.get(index)
    if ptr is None:
        with _status_lock:                  # one word for all threads that come here first
            ptr = _status_ptrs.get(index)
            if ptr is None:
                word = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
                torch.cuda.current_stream(word.device).synchronize()    # zeroed before any other stream's kernel sees it
                _status_words[index] = word
                ptr = _status_ptrs[index] = word.data_ptr()
    return ptr


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
_INT32_MAX = 2 ** 31 - 1
_HALF_OR_F32 = (torch.float16, torch.bfloat16, torch.float32)


def _shape(t, shape, name):
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _plain(t, dim, index, dtype):
    """Whether _dev(t, ...) would pass."""
    return t.dim() == dim and t.dtype is dtype and t.get_device() == index and (t.stride(-1) == 1 or t.shape[-1] <= 1)


def _matrix(t, name, index, dtype):
    """(pointer, rows, columns, row stride) of a matrix with rows that do not overlap; a stride that the row count leaves
    without meaning is taken as the row length."""
    if t.dim() != 2 or t.dtype is not dtype or t.get_device() != index:
        _dev(t, name, 2, index, (dtype,))
    n, k = t.shape
    ld, one = t.stride()
    if n <= 1:
        ld = max(k, 1)
    if ld < k or (one != 1 and k > 1):
        _rows_ok(_dev(t, name, 2, index, (dtype,)), name)
    return t.data_ptr(), n, k, ld


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
    dt = x.dtype
    if dt not in _HALF or not x.is_cuda:
        _dev(x, "x", 2, None, _HALF)
    index = x.get_device()
    if _current_device() != index:
        with torch.cuda.device(index):
            return linear(x, w, bias, activation, residual, save_pre, out_dtype, out)
    xp, M, K, ldx = _matrix(x, "x", index, dt)
    wp, N, wk, ldw = _matrix(w, "w", index, dt)
    if wk != K:
        raise ValueError(f"w must be [N, {K}], got {tuple(w.shape)}")
    if N < 1 or K < 1:
        raise ValueError("w must not be empty")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    bp = None
    if bias is not None:
        if not _plain(bias, 1, index, dt) or bias.shape[0] != N:
            _shape(_dev(bias, "bias", 1, index, (dt,)), (N,), "bias")
        bp = bias.data_ptr()
    odt, rp, ldr = out_dtype or dt, None, 0
    if residual is not None:
        rdt = residual.dtype
        if rdt is not dt and rdt is not torch.float32:
            _dev(residual, "residual", 2, index, (dt, torch.float32))
        if out_dtype is None:
            odt = rdt
        elif rdt is not odt:
            raise TypeError(f"residual must have the output's type {odt}, got {rdt}")
        rp, rm, rn, ldr = _matrix(residual, "residual", index, rdt)
        if rm != M or rn != N:
            _shape(residual, (M, N), "residual")
    if odt is not dt and odt is not torch.float32:
        raise TypeError(f"out_dtype must be {dt} or torch.float32, got {odt}")
    if out is None:
        y, ldy = x.new_empty((M, N), dtype=odt), N
        yp = y.data_ptr()
    else:
        y = out
        yp, om, on, ldy = _matrix(out, "out", index, odt)
        if om != M or on != N:
            _shape(out, (M, N), "out")
    pre = x.new_empty((M, N)) if save_pre else None
    if M:
        need = _query("pmg_linear_workspace_bytes", M, N, K, (xp | 2 * ldx) & 15, (wp | 2 * ldw) & 15) if M > 32 else 0
        ws = x.new_empty(need, dtype=torch.uint8) if need else None
        _call("pmg_linear", xp, ldx, wp, ldw, _DTYPES[dt], M, N, K, bp, act, rp, ldr, odt is torch.float32, yp, ldy,
              pre.data_ptr() if save_pre else None, N, ws.data_ptr() if need else None, need, _status(index),
              _current_stream(index))
    return (y, pre) if save_pre else y


def linear_grad(dy, x, w, pre=None, activation: str = "none", bias_grad: bool = True, input_grad: bool = True,
                weight_grad: bool = True):
    """Gradients (dx, dw, dbias) of linear() for dy [M, N], the gradient of its output, in x's type (dy too); None for
    one that is not asked for.  pre: the second output of linear(..., save_pre=True), needed unless the activation is
    "none".  The residual's gradient is dy itself."""
    dt = x.dtype
    if dt not in _HALF or not x.is_cuda:
        _dev(x, "x", 2, None, _HALF)
    index = x.get_device()
    if _current_device() != index:
        with torch.cuda.device(index):
            return linear_grad(dy, x, w, pre, activation, bias_grad, input_grad, weight_grad)
    xp, M, K, ldx = _matrix(x, "x", index, dt)
    wp, N, wk, ldw = _matrix(w, "w", index, dt)
    yp, ym, yn, ldy = _matrix(dy, "dy", index, dt)
    if wk != K or N < 1 or K < 1:
        raise ValueError(f"w must be [N, {K}], got {tuple(w.shape)}")
    if ym != M or yn != N:
        _shape(dy, (M, N), "dy")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    pp, ldp = None, 0
    if act:
        if pre is None:
            raise ValueError("pre (linear(..., save_pre=True)) is needed for an activation's gradient")
        pp, pm, pn, ldp = _matrix(pre, "pre", index, dt)
        if pm != M or pn != N:
            _shape(pre, (M, N), "pre")
    dx = x.new_empty((M, K)) if input_grad else None
    dw = x.new_empty((N, K)) if weight_grad else None
    db = x.new_empty(N) if bias_grad else None
    need = _query("pmg_linear_grad_workspace_bytes", M, N, K, act, (yp | 2 * ldy) & 15,
                  (xp | 2 * ldx) & 15 if weight_grad else 0, (wp | 2 * ldw) & 15 if input_grad else 0, int(bias_grad))
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    _call("pmg_linear_grad", yp, ldy, xp, ldx, wp, ldw, _DTYPES[dt], M, N, K, pp, ldp, act,
          dx.data_ptr() if input_grad else None, K, dw.data_ptr() if weight_grad else None, K,
          db.data_ptr() if bias_grad else None, ws.data_ptr() if need else None, need, _status(index),
          _current_stream(index))
    return dx, dw, db


# ----------------------------------------------------------------------------------------------------------------- #
# Norm of queries and keys with the position rotation
# ----------------------------------------------------------------------------------------------------------------- #
def _heads(t, name, index, dtype, T, H, D):
    """(pointer, token stride, head stride) of [T, H, D]."""
    if t.dtype is dtype and t.get_device() == index and t.shape == (T, H, D):
        st, sh, one = t.stride()
        if one == 1 or D <= 1:
            return t.data_ptr(), st, sh
    _shape(_dev(t, name, 3, index, (dtype,)), (T, H, D), name)
    return t.data_ptr(), *t.stride()[:2]


def _angles(cos, sin, positions, T, D, index):
    """(cos, sin, pairs, places, positions) as the entry points take them."""
    for t, name in ((cos, "cos"), (sin, "sin")):
        if t.dtype is not torch.float32 or t.get_device() != index or t.dim() != 2:
            _dev(t, name, 2, index, (torch.float32,))
    places, half = cos.shape
    if sin.shape != (places, half):
        _shape(sin, cos.shape, "sin")
    if 2 * half > D:
        raise ValueError(f"cos and sin rotate {2 * half} values of heads of {D}")
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous")
    if half and T and places == 0:
        raise ValueError("cos and sin must not be empty")
    if positions is not None:
        return cos.data_ptr(), sin.data_ptr(), half, places, _words(positions, "positions", T, index)
    if T > places and half:
        raise ValueError(f"{T} tokens without positions need as many rows of cos and sin, got {places}")
    return cos.data_ptr(), sin.data_ptr(), half, places, None


def _weight(w, name, D, index):
    if w is None:
        return None
    return _words(w, name, D, index, torch.float32)


def _qk(q, k):
    dt = q.dtype
    index = q.get_device()
    if dt not in _DTYPES or index < 0 or q.dim() != 3 or (q.stride(2) != 1 and q.shape[2] > 1):
        _dev(q, "q", 3, None, _HALF_OR_F32)
    if not _plain(k, 3, index, dt):
        _dev(k, "k", 3, index, (dt,))
    T, Hq, D = q.shape
    kt, Hk, kd = k.shape
    if kt != T or kd != D:
        raise ValueError(f"k must be [{T}, heads, {D}], got {tuple(k.shape)}")
    if D < 1 or D > 256:
        raise ValueError(f"heads hold 1 to 256 values, got {D}")
    return index, dt, T, Hq, Hk, D


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6, interleaved: bool = False,
                 out=None):
    """Queries [T, Hq, D] and keys [T, Hk, D] (fp32, fp16 or bf16), each head divided by its root mean square and
    multiplied by the weight ([D] fp32 or None), then its first 2 * cos.shape[1] values rotated by the angles of the
    token's position: cos, sin [places, pairs] fp32; positions [T] int32 (None: 0, 1, 2, ...).  Pairs are (i, i +
    pairs), or (2i, 2i + 1) when interleaved.  out: a pair of tensors to write to, which may be q and k themselves or
    rows of a cache.  Returns (q, k)."""
    index, dt, T, Hq, Hk, D = _qk(q, k)
    if _current_device() != index:
        with torch.cuda.device(index):
            return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, out)
    cp, sp, half, places, pp = _angles(cos, sin, positions, T, D, index)
    qh, kh = (q.data_ptr(), *q.stride()[:2]), (k.data_ptr(), *k.stride()[:2])
    if out is None:
        qo, ko = q.new_empty((T, Hq, D)), q.new_empty((T, Hk, D))
        qoh, koh = (qo.data_ptr(), Hq * D, D), (ko.data_ptr(), Hk * D, D)
    else:
        qo, ko = out
        qoh, koh = _heads(qo, "out[0]", index, dt, T, Hq, D), _heads(ko, "out[1]", index, dt, T, Hk, D)
    _call("pmg_qk_norm_rope", *qh, *kh, _DTYPES[dt], T, Hq, Hk, D, 2 * half, _weight(q_weight, "q_weight", D, index),
          _weight(k_weight, "k_weight", D, index), cp, sp, places, pp, eps, bool(interleaved), *qoh, *koh,
          _status(index), _current_stream(index))
    return qo, ko


def qk_norm_rope_grad(dq, dk, q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6,
                      interleaved: bool = False):
    """Gradients (q, k, q_weight, k_weight) of qk_norm_rope() for the gradients dq, dk of its outputs and its inputs
    q, k; the weights' in fp32, None where there is no weight."""
    index, dt, T, Hq, Hk, D = _qk(q, k)
    if _current_device() != index:
        with torch.cuda.device(index):
            return qk_norm_rope_grad(dq, dk, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    cp, sp, half, places, pp = _angles(cos, sin, positions, T, D, index)
    gq, gk = q.new_empty((T, Hq, D)), q.new_empty((T, Hk, D))
    gqw = q.new_empty(D, dtype=torch.float32) if q_weight is not None else None
    gkw = q.new_empty(D, dtype=torch.float32) if k_weight is not None else None
    need, ws = 0, None
    if q_weight is not None or k_weight is not None:
        need = _query("pmg_qk_norm_rope_grad_workspace_bytes", D)
        ws = q.new_empty(need, dtype=torch.uint8)
    qs, ks = (T, Hq, D), (T, Hk, D)
    _call("pmg_qk_norm_rope_grad", *_heads(dq, "dq", index, dt, *qs), *_heads(dk, "dk", index, dt, *ks),
          *_heads(q, "q", index, dt, *qs), *_heads(k, "k", index, dt, *ks), _DTYPES[dt], T, Hq, Hk, D, 2 * half,
          _weight(q_weight, "q_weight", D, index), _weight(k_weight, "k_weight", D, index), cp, sp, places, pp, eps,
          bool(interleaved), gq.data_ptr(), Hq * D, D, gk.data_ptr(), Hk * D, D,
          gqw.data_ptr() if gqw is not None else None, gkw.data_ptr() if gkw is not None else None,
          ws.data_ptr() if need else None, need, _status(index), _current_stream(index))
    return gq, gk, gqw, gkw


# ----------------------------------------------------------------------------------------------------------------- #
# Attention over packed documents
# ----------------------------------------------------------------------------------------------------------------- #
def _aligned_heads(t, name, T, H, D, index, dt):
    """(pointer, token stride, head stride) of [T, H, D] on 16-byte boundaries."""
    p, st, sh = _heads(t, name, index, dt, T, H, D)
    if H <= 1:
        sh = D
    if T <= 1:
        st = H * D if sh == D else (st + 7) // 8 * 8
    if (p | 2 * st | 2 * sh) & 15:
        raise ValueError(f"{name}: heads must start on 16-byte boundaries (strides in multiples of 8 values)")
    return p, st, sh


def _words(t, name, n, index, dtype=torch.int32):
    """The pointer of a vector of n values."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        _shape(_dev(t, name, 1, index, (dtype,)), (n,), name)
    return t.data_ptr()


def _mask_words(cu_q, cu_k, k_len, prefix, slopes, docs, Hq, index):
    return (_words(cu_q, "cu_q", docs + 1, index), _words(cu_k, "cu_k", docs + 1, index),
            None if k_len is None else _words(k_len, "k_len", docs, index),
            None if prefix is None else _words(prefix, "prefix", docs, index),
            None if slopes is None else _words(slopes, "slopes", Hq, index, torch.float32))


def _attention_shapes(q, k):
    dt = q.dtype
    index = q.get_device()
    if dt not in _HALF or index < 0 or q.dim() != 3:
        _dev(q, "q", 3, None, _HALF)
    if k.dtype is not dt or k.dim() != 3:
        _dev(k, "k", 3, index, (dt,))
    Tq, Hq, D = q.shape
    Tk, Hk, kd = k.shape
    if kd != D or Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError(f"k must be [keys, heads, {D}] with a number of heads that divides {Hq}, got {tuple(k.shape)}")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"heads must hold a multiple of 8 values, 8 to 128, got {D}")
    return index, dt, Tq, Tk, Hq, Hk, D


def _documents(cu_q):
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q must hold the documents' offsets, the total last")
    return cu_q.shape[0] - 1


def _score(scale, D, softcap, causal, prefix, max_q, max_k):
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf") or not 0.0 <= softcap < float("inf"):
        raise ValueError("scale must be positive and softcap not negative, both finite")
    if not (0 <= max_q <= _INT32_MAX and 0 <= max_k <= _INT32_MAX):
        raise ValueError("max_q and max_k must be 0 to 2^31 - 1")
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

    Returns (o [Tq, Hq, D], lse [Hq, Tq] fp32).  Rows that see no key give 0 and -inf; rows of no document (in front of
    cu_q[0] and from the last offset on) are not written.  max_q * Hq / Hk <= 16 (token by token) takes the kernel that
    reads the keys once for all rows."""
    index, dt, Tq, Tk, Hq, Hk, D = _attention_shapes(q, k)
    if _current_device() != index:
        with torch.cuda.device(index):
            return attention(q, k, v, cu_q, cu_k, max_q, max_k, scale, causal, prefix, softcap, slopes, k_len, out)
    docs = _documents(cu_q)
    scale = _score(scale, D, softcap, causal, prefix, max_q, max_k)
    words = _mask_words(cu_q, cu_k, k_len, prefix, slopes, docs, Hq, index)
    qh, kh = _aligned_heads(q, "q", Tq, Hq, D, index, dt), _aligned_heads(k, "k", Tk, Hk, D, index, dt)
    vh = _aligned_heads(v, "v", Tk, Hk, D, index, dt)
    if out is None:
        o = q.new_empty((Tq, Hq, D))
        oh = (o.data_ptr(), Hq * D, D)
    else:
        o, oh = out, _aligned_heads(out, "out", Tq, Hq, D, index, dt)
    lse = q.new_empty((Hq, Tq), dtype=torch.float32)
    if Tq:
        need = _query("pmg_attention_workspace_bytes", docs, Hq, Hk, D, max_q, max_k) if max_q * Hq <= 16 * Hk else 0
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        _call("pmg_attention", *qh, *kh, *vh, _DTYPES[dt], Tq, Tk, Hq, Hk, D, words[0], words[1], words[2], docs, max_q,
              max_k, scale, bool(causal), words[3], softcap, words[4], *oh, lse.data_ptr(),
              ws.data_ptr() if need else None, need, _status(index), _current_stream(index))
    return o, lse


def attention_grad(do, o, lse, q, k, v, cu_q, cu_k, max_q: int, max_k: int, scale: float | None = None,
                   causal: bool = False, prefix=None, softcap: float = 0.0, slopes=None, k_len=None):
    """Gradients (dq, dk, dv) of attention() for do, the gradient of its output: o and lse are what it returned, the
    rest its arguments.  The slopes are constants of the score and get no gradient.  Key rows behind k_len get zeros."""
    index, dt, Tq, Tk, Hq, Hk, D = _attention_shapes(q, k)
    if _current_device() != index:
        with torch.cuda.device(index):
            return attention_grad(do, o, lse, q, k, v, cu_q, cu_k, max_q, max_k, scale, causal, prefix, softcap, slopes,
                                  k_len)
    docs = _documents(cu_q)
    scale = _score(scale, D, softcap, causal, prefix, max_q, max_k)
    words = _mask_words(cu_q, cu_k, k_len, prefix, slopes, docs, Hq, index)
    if not _plain(lse, 2, index, torch.float32) or lse.shape != (Hq, Tq):
        _shape(_dev(lse, "lse", 2, index, (torch.float32,)), (Hq, Tq), "lse")
    if not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    qs, ks = (Tq, Hq, D), (Tk, Hk, D)
    heads = (*_aligned_heads(do, "do", *qs, index, dt), *_aligned_heads(o, "o", *qs, index, dt), lse.data_ptr(),
             *_aligned_heads(q, "q", *qs, index, dt), *_aligned_heads(k, "k", *ks, index, dt),
             *_aligned_heads(v, "v", *ks, index, dt))
    dq, dk, dv = q.new_empty(qs), q.new_empty(ks), q.new_empty(ks)
    need = _query("pmg_attention_grad_workspace_bytes", Tq, Hq)
    ws = q.new_empty(need, dtype=torch.uint8)
    st = (Hk * D, D)
    _call("pmg_attention_grad", *heads, _DTYPES[dt], Tq, Tk, Hq, Hk, D, words[0], words[1], words[2], docs, scale,
          bool(causal), words[3], softcap, words[4], dq.data_ptr(), Hq * D, D, dk.data_ptr(), *st, dv.data_ptr(), *st,
          ws.data_ptr(), need, _status(index), _current_stream(index))
    return dq, dk, dv
