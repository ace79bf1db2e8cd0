"""Operators of an encoder block on device tensors: layer norm (csrc/ln.hip), differential attention (csrc/diffattn.hip) and
the Newton-Schulz orthogonalisation of a Muon update (csrc/newton_schulz.hip).

``layer_norm`` and ``diff_attention`` are differentiable; their ``*_fwd`` / ``*_bwd`` forms are the two passes without
autograd, for serving, for hand-written training steps and for HIP graphs (a captured autograd backward is refused: replay
one that was captured with the ``*_bwd`` forms).  All of them run on the current stream of their tensors' device, take
their workspace from torch's allocator at each call (a captured graph so keeps its own) and never synchronise.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from ._lib import DiffAttn, NsMat, call, query

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
NS_COEFFS = (3.4445, -4.7750, 2.0315)


class _On:
    """The device of the tensors as the current one, where it is not already."""

    __slots__ = ("idx", "prev")

    def __init__(self, t):
        self.idx = t.device.index

    def __enter__(self):
        cur = torch.cuda.current_device()
        self.prev = cur if cur != self.idx else None
        if self.prev is not None:
            torch.cuda.set_device(self.idx)
        return torch._C._cuda_getCurrentRawStream(self.idx)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)


def _device(name, *tensors):
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"{name}: device tensors, got {dev}")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: tensors on {dev} and {t.device}")


def _no_capture(name):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name}: the autograd backward cannot be captured into a graph; capture {name}_bwd")


# ---------------------------------------------------------------------------------------------- layer norm
def _rows(t):
    """(rows, width) view of t without a copy where its leading axes have one stride, else of a copy."""
    n = t.shape[-1]
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.stride(-1) != 1 and n > 1:
        t = t.contiguous()
    try:
        r = t.view(-1, n)
    except RuntimeError:
        r = t.contiguous().view(-1, n)
    if r.shape[0] > 1 and r.stride(0) < 0:
        r = r.contiguous()
    return r


def _check_norm(name, x, weight, bias):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: rows of at least one element, got {tuple(x.shape)}")
    n = x.shape[-1]
    if x.dtype not in _TYPES:
        raise TypeError(f"{name}: float32, bfloat16 or float16 rows, got {x.dtype}")
    for w, what in ((weight, "weight"), (bias, "bias")):
        if w is None:
            continue
        if tuple(w.shape) != (n,):
            raise ValueError(f"{name}: {what} of shape {(n,)}, got {tuple(w.shape)}")
        if w.dtype != weight.dtype or w.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"{name}: {what} in float32 or the rows' type, weight and bias alike, got {w.dtype}")


def layer_norm_fwd(x, weight, bias=None, eps=1e-5):
    """(y, mean, rstd) of y = (x - mean) * rstd * weight + bias over the last axis; mean and rstd (one a row, float32) are
    what ``layer_norm_bwd`` needs.  x: (..., N) float32 / bfloat16 / float16; weight, bias: (N,) float32 or x's type."""
    _check_norm("layer_norm", x, weight, bias)
    _device("layer_norm", x, weight, bias)
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps >= 0, got {eps}")
    n = x.shape[-1]
    r = _rows(x)
    m = r.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stat = torch.empty((2, m), dtype=torch.float32, device=x.device)
    w = weight.contiguous()
    b = bias.contiguous() if bias is not None else None
    if m:
        with _On(x) as st:
            call("ctr_ln_fwd", r.data_ptr(), r.stride(0), m, n, w.data_ptr(), b.data_ptr() if b is not None else None,
                 float(eps), y.data_ptr(), n, stat.data_ptr(), stat.data_ptr() + 4 * m, _TYPES[x.dtype],
                 _TYPES[w.dtype], st)
    return y, stat[0], stat[1]


def layer_norm_bwd(dy, x, mean, rstd, weight, bias=True):
    """(dx, dweight, dbias) of ``layer_norm_fwd``; dbias is None with ``bias=False``.  The weight gradients are the sums over
    all rows, in the weight's type."""
    _check_norm("layer_norm_bwd", x, weight, None)
    _device("layer_norm_bwd", dy, x, mean, rstd, weight)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"layer_norm_bwd: dy of x's shape and type, got {tuple(dy.shape)} {dy.dtype}")
    n = x.shape[-1]
    r, g = _rows(x), _rows(dy)
    m = r.shape[0]
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if t.numel() != m or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"layer_norm_bwd: {what} as layer_norm_fwd gave it: {m} float32 values")
    w = weight.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty_like(w)
    db = torch.empty_like(w) if bias else None
    with _On(x) as st:
        size = query("ctr_ln_bwd_ws_size", m, n)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        call("ctr_ln_bwd", g.data_ptr(), g.stride(0), r.data_ptr(), r.stride(0), mean.data_ptr(), rstd.data_ptr(),
             w.data_ptr(), m, n, dx.data_ptr(), n, dw.data_ptr(), db.data_ptr() if bias else None,
             ws.data_ptr() if size else None, size, _TYPES[x.dtype], _TYPES[w.dtype], st)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_capture("layer_norm")
        x, mean, rstd, weight = ctx.saved_tensors
        dx, dw, db = layer_norm_bwd(dy, x, mean, rstd, weight, ctx.bias)
        return dx, dw, db, None


def layer_norm(x, weight, bias=None, eps=1e-5):
    """Differentiable layer norm over the last axis (see ``layer_norm_fwd``)."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ---------------------------------------------------------------------------------------------- differential attention
def _aligned(t):
    """t, or a copy of it where its rows cannot be read 16 bytes at a time."""
    if t.numel() and (t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:-1], t.shape)
                                                                      if n > 1)):
        return t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def _strides(t):
    """Element strides of the leading axes; an axis of one element has none that matters."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


def _lens(name, lens, b, dev):
    if lens is None:
        return None
    if lens.dtype != torch.int32 or tuple(lens.shape) != (b,) or lens.device != dev:
        raise ValueError(f"{name}: {b} int32 lengths on {dev}, got {tuple(lens.shape)} {lens.dtype} on {lens.device}")
    return lens.contiguous()


def _attn_args(name, q, k, v, lam, causal, scale, q_lens, kv_lens):
    if q.dim() != 5 or q.shape[3] != 2:
        raise ValueError(f"{name}: q of shape (B, T, H, 2, D), got {tuple(q.shape)}")
    B, T, H, _, D = q.shape
    if k.dim() != 5 or k.shape[0] != B or k.shape[3] != 2 or k.shape[4] != D:
        raise ValueError(f"{name}: k of shape ({B}, S, Hkv, 2, {D}), got {tuple(k.shape)}")
    S, Hkv = k.shape[1], k.shape[2]
    if tuple(v.shape) != (B, S, Hkv, 2 * D):
        raise ValueError(f"{name}: v of shape {(B, S, Hkv, 2 * D)}, got {tuple(v.shape)}")
    if D not in (32, 64, 128):
        raise NotImplementedError(f"{name}: maps of width 32, 64 or 128, got {D}")
    if H < 1 or Hkv < 1 or H % Hkv:
        raise ValueError(f"{name}: {H} query heads over {Hkv} key heads")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name}: bfloat16 or float16, got {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{name}: q, k and v of one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if tuple(lam.shape) != (H,) or lam.dtype != torch.float32:
        raise ValueError(f"{name}: lam of {H} float32 values, got {tuple(lam.shape)} {lam.dtype}")
    _device(name, q, k, v, lam)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{name}: scale > 0, got {scale}")
    q, k, v, lam = _aligned(q), _aligned(k), _aligned(v), lam.contiguous()
    ql, kl = _lens(name + " q_lens", q_lens, B, q.device), _lens(name + " kv_lens", kv_lens, B, q.device)
    a = DiffAttn()
    a.q, a.k, a.v, a.lam = q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr()
    a.q_lens, a.kv_lens = ql.data_ptr() if ql is not None else None, kl.data_ptr() if kl is not None else None
    a.q_sb, a.q_st, a.q_sh, a.q_sc = _strides(q)
    a.k_sb, a.k_ss, a.k_sh, a.k_sc = _strides(k)
    a.v_sb, a.v_ss, a.v_sh = _strides(v)
    a.scale, a.B, a.T, a.S, a.H, a.Hkv, a.D = scale, B, T, S, H, Hkv, D
    a.causal, a.type = int(bool(causal)), _TYPES[q.dtype]
    return a, (q, k, v, lam, ql, kl)


def diff_attention_fwd(q, k, v, lam, causal=False, scale=None, q_lens=None, kv_lens=None, save=True):
    """(out, saved): out = (softmax(q1 k1^T scale) - lam softmax(q2 k2^T scale)) v, of shape (B, T, H, 2 D).

    q: (B, T, H, 2, D) -- the two maps' queries of a head side by side; k: (B, S, Hkv, 2, D); v: (B, S, Hkv, 2 D); H a
    multiple of Hkv (key head j serves the query heads j H / Hkv ...); bfloat16 or float16, D in {32, 64, 128}; lam: (H,)
    float32.  Any strides with the last axis contiguous and 16-byte aligned rows are read in place (a slice of a cache),
    others from a copy.  scale: 1 / sqrt(D) unless given.  q_lens / kv_lens: (B,) int32 device tensors, the valid
    positions and keys of each sequence, held to [0, T] / [0, S]; what stands behind them does not count.  causal: position t
    sees the keys up to t + kv_len - q_len, so one new token (T = 1) sees its whole cache.  Rows that see no key, and
    positions behind q_lens, are zeros.  ``saved`` is for ``diff_attention_bwd`` (None with ``save=False``)."""
    a, keep = _attn_args("diff_attention", q, k, v, lam, causal, scale, q_lens, kv_lens)
    out = torch.empty((a.B, a.T, a.H, 2 * a.D), dtype=q.dtype, device=q.device)
    saved = None
    a.o = out.data_ptr()
    if save:
        parts = torch.empty((2, *out.shape), dtype=q.dtype, device=q.device)     # the second map's, out's remainder
        stat = torch.empty((2, a.B * a.H * a.T), dtype=torch.float32, device=q.device)
        a.o2, a.ol, a.stat = parts.data_ptr(), parts.data_ptr() + 2 * out.numel(), stat.data_ptr()
        saved = (parts, stat)
    if out.numel():
        with _On(q) as st:
            size = query("ctr_diffattn_fwd_ws_size", C.byref(a))
            ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
            call("ctr_diffattn_fwd", C.byref(a), ws.data_ptr() if size else None, size, st)
    return out, saved


def diff_attention_bwd(dout, q, k, v, lam, out, saved, causal=False, scale=None, q_lens=None, kv_lens=None):
    """(dq, dk, dv, dlam) of ``diff_attention_fwd``, given its out and saved and the same other arguments."""
    a, keep = _attn_args("diff_attention_bwd", q, k, v, lam, causal, scale, q_lens, kv_lens)
    shape = (a.B, a.T, a.H, 2 * a.D)
    if saved is None:
        raise ValueError("diff_attention_bwd: the forward ran with save=False")
    parts, stat = saved
    for t, what in ((dout, "dout"), (out, "out")):
        if tuple(t.shape) != shape or t.dtype != q.dtype:
            raise ValueError(f"diff_attention_bwd: {what} of shape {shape} {q.dtype}, got {tuple(t.shape)} {t.dtype}")
    if tuple(parts.shape) != (2, *shape) or parts.dtype != q.dtype or not parts.is_contiguous() or \
            tuple(stat.shape) != (2, a.B * a.H * a.T) or stat.dtype != torch.float32 or not stat.is_contiguous():
        raise ValueError("diff_attention_bwd: saved as diff_attention_fwd gave it")
    _device("diff_attention_bwd", q, dout, out, parts, stat)
    dout, out = _aligned(dout), _aligned(out.contiguous())
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    dv = torch.empty(v.shape, dtype=q.dtype, device=q.device)
    dlam = torch.empty(a.H, dtype=torch.float32, device=q.device)
    a.o, a.stat = out.data_ptr(), stat.data_ptr()
    a.o2, a.ol = parts.data_ptr(), parts.data_ptr() + 2 * out.numel()
    with _On(q) as st:
        size = query("ctr_diffattn_bwd_ws_size", C.byref(a))
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        call("ctr_diffattn_bwd", C.byref(a), dout.data_ptr(), *_strides(dout), dq.data_ptr(), dk.data_ptr(),
             dv.data_ptr(), dlam.data_ptr(), ws.data_ptr() if size else None, size, st)
    return dq, dk, dv, dlam


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, causal, scale, q_lens, kv_lens):
        out, saved = diff_attention_fwd(q, k, v, lam, causal, scale, q_lens, kv_lens)
        ctx.save_for_backward(q, k, v, lam, out, q_lens, kv_lens, *saved)
        ctx.args = (causal, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _no_capture("diff_attention")
        q, k, v, lam, out, q_lens, kv_lens, *saved = ctx.saved_tensors
        grads = diff_attention_bwd(dout, q, k, v, lam, out, tuple(saved), *ctx.args, q_lens, kv_lens)
        return (*grads, None, None, None, None)


def diff_attention(q, k, v, lam, causal=False, scale=None, q_lens=None, kv_lens=None):
    """Differentiable differential attention (see ``diff_attention_fwd``)."""
    return _DiffAttention.apply(q, k, v, lam, causal, scale, q_lens, kv_lens)


# ---------------------------------------------------------------------------------------------- Newton-Schulz
@torch.no_grad()
def newton_schulz(mats, steps=5, coeffs=NS_COEFFS, eps=1e-7):
    """Orthogonalised matrices: X = G / (||G||_F + eps), then ``steps`` times X <- (a I + b A + c A^2) X with A = X X^T (of
    the transpose when G has more rows than columns).  mats: a matrix, a batch (..., m, n) or a list of matrices of any
    shapes and one type (float32, bfloat16, float16); the result likewise.  Computed to float32's accuracy whatever the
    type.  Coefficients under which a singular value could leave [0, 7.5] are refused."""
    single = isinstance(mats, torch.Tensor)
    lst = [mats] if single else list(mats)
    if not lst:
        return []
    for t in lst:
        if t.dim() < 2 or (not single and t.dim() != 2):
            raise ValueError(f"newton_schulz: matrices, got a shape of {tuple(t.shape)}")
        if t.dtype not in _TYPES or t.dtype != lst[0].dtype:
            raise TypeError(f"newton_schulz: one of float32, bfloat16, float16 for all, got {t.dtype}")
    _device("newton_schulz", *lst)
    if not 1 <= int(steps) <= 64:
        raise ValueError(f"newton_schulz: steps in [1, 64], got {steps}")
    out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in lst]
    pairs = []
    for t, o in zip(lst, out):
        if t.numel() == 0:
            continue
        m, n = t.shape[-2:]
        if (t.stride(-1) != 1 and n > 1) or (t.stride(-2) < n and m > 1):
            t = t.contiguous()
        if t.dim() == 2:
            pairs.append((t, o))
        else:
            try:
                flat = t.view(-1, m, n)
            except RuntimeError:
                flat = t.contiguous().view(-1, m, n)
            pairs += list(zip(flat.unbind(0), o.view(-1, m, n).unbind(0)))
    if pairs:
        arr = (NsMat * len(pairs))()
        for e, (t, o) in zip(arr, pairs):
            e.src, e.dst, e.rows, e.cols = t.data_ptr(), o.data_ptr(), t.shape[0], t.shape[1]
            e.ld_src, e.ld_dst = max(t.stride(0), t.shape[1]), o.shape[1]
        a, b, c = (float(v) for v in coeffs)
        with _On(lst[0]) as st:
            size = query("ctr_newton_schulz_ws_size", arr, len(pairs))
            ws = torch.empty(size, dtype=torch.uint8, device=lst[0].device) if size else None
            call("ctr_newton_schulz", arr, len(pairs), int(steps), a, b, c, float(eps), _TYPES[lst[0].dtype],
                 ws.data_ptr() if size else None, size, st)
    return out[0] if single else out
