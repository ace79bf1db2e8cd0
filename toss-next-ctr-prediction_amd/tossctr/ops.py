"""Operators of an encoder block on device tensors: layer norm (csrc/ln.hip), differential attention (csrc/diffattn.hip) and
the Newton-Schulz orthogonalisation of a Muon update (csrc/newton_schulz.hip).

``layer_norm`` and ``diff_attention`` are differentiable; their ``*_fwd`` / ``*_bwd`` forms are the two passes without
autograd, for serving, for hand-written training steps and for HIP graphs: a differentiable call under capture is refused, and
the backward pass of an eager one is not to be captured (torch's engine ties it to the eager call's stream).  All of them run on
the current stream of their tensors' device, take their workspace from torch's allocator at each call (a captured graph so keeps
its own) and never synchronise.
"""
from __future__ import annotations

import array
import ctypes as C
import math

import torch

from . import _lib
from ._lib import DiffAttn, NsMat, call, query

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
NS_COEFFS = (3.4445, -4.7750, 2.0315)


_raw_stream = torch._C._cuda_getCurrentRawStream
_get_device = torch._C._cuda_getDevice


def _launch(t, name, *args):
    """call(name, *args, stream) with t's device as the current one and its current stream."""
    idx = t.get_device()
    prev = _get_device()
    if prev == idx:
        call(name, *args, _raw_stream(idx))
        return
    torch.cuda.set_device(idx)
    try:
        call(name, *args, _raw_stream(idx))
    finally:
        torch.cuda.set_device(prev)


def _device(name, *tensors):
    idx = tensors[0].get_device()
    if idx < 0:
        raise ValueError(f"{name}: device tensors, got {tensors[0].device}")
    for t in tensors[1:]:
        if t is not None and t.get_device() != idx:
            raise ValueError(f"{name}: tensors on {tensors[0].device} and {t.device}")


def _no_capture(name, *tensors):
    # torch's engine runs a node on the stream of its forward pass and waits for the leaves' own: with an eager graph of the same
    # leaves alive, a captured backward waits for a stream outside the capture, which ends the process
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors) and \
            torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name}: no differentiable call under graph capture; capture {name}_fwd and {name}_bwd")


# ---------------------------------------------------------------------------------------------- layer norm
def _rows(t):
    """t or a copy of it, and the stride of its rows, where its leading axes have one stride."""
    n = t.shape[-1]
    if t.is_contiguous():
        return t, n
    if t.stride(-1) == 1 or n == 1:
        try:
            r = t.view(-1, n)
            return t, r.stride(0) if r.shape[0] > 1 else n
        except RuntimeError:
            pass
    return t.contiguous(), n


def _check_norm(name, x, weight, bias):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: rows of at least one element, got {tuple(x.shape)}")
    n, dt, wt = x.shape[-1], x.dtype, weight.dtype
    if dt not in _TYPES:
        raise TypeError(f"{name}: float32, bfloat16 or float16 rows, got {dt}")
    if weight.dim() != 1 or weight.shape[0] != n:
        raise ValueError(f"{name}: weight of shape {(n,)}, got {tuple(weight.shape)}")
    if wt is not torch.float32 and wt is not dt:
        raise TypeError(f"{name}: weight in float32 or the rows' type, got {wt}")
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != n:
            raise ValueError(f"{name}: bias of shape {(n,)}, got {tuple(bias.shape)}")
        if bias.dtype is not wt:
            raise TypeError(f"{name}: bias in float32 or the rows' type, as the weight, got {bias.dtype}")
    return n, _TYPES[dt], _TYPES[wt]


def layer_norm_fwd(x, weight, bias=None, eps=1e-5):
    """(y, mean, rstd) of y = (x - mean) * rstd * weight + bias over the last axis; mean and rstd (one a row, float32) are
    what ``layer_norm_bwd`` needs.  x: (..., N) float32 / bfloat16 / float16; weight, bias: (N,) float32 or x's type."""
    n, xt, wt = _check_norm("layer_norm", x, weight, bias)
    _device("layer_norm", x, weight, bias)
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps >= 0, got {eps}")
    m = x.numel() // n
    r, ld = _rows(x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean, rstd = x.new_empty((2, m), dtype=torch.float32).unbind(0)
    if m:
        w = weight.contiguous()
        b = bias.contiguous() if bias is not None else None
        _launch(x, "ctr_ln_fwd", r.data_ptr(), ld, m, n, w.data_ptr(), None if b is None else b.data_ptr(), eps,
                y.data_ptr(), n, mean.data_ptr(), rstd.data_ptr(), xt, wt)
    return y, mean, rstd


def layer_norm_bwd(dy, x, mean, rstd, weight, bias=True):
    """(dx, dweight, dbias) of ``layer_norm_fwd``; dbias is None with ``bias=False``.  The weight gradients are the sums over
    all rows, in the weight's type."""
    n, xt, wt = _check_norm("layer_norm_bwd", x, weight, None)
    _device("layer_norm_bwd", dy, x, mean, rstd, weight)
    if dy.shape != x.shape or dy.dtype is not x.dtype:
        raise ValueError(f"layer_norm_bwd: dy of x's shape and type, got {tuple(dy.shape)} {dy.dtype}")
    m = x.numel() // n
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if t.numel() != m or t.dtype is not torch.float32 or not t.is_contiguous():
            raise ValueError(f"layer_norm_bwd: {what} as layer_norm_fwd gave it: {m} float32 values")
    (r, ld), (g, ldg) = _rows(x), _rows(dy)
    w = weight.contiguous()
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dw = torch.empty_like(w)
    db = torch.empty_like(w) if bias else None
    size = query("ctr_ln_bwd_ws_size", m, n)
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    _launch(x, "ctr_ln_bwd", g.data_ptr(), ldg, r.data_ptr(), ld, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), m, n,
            dx.data_ptr(), n, dw.data_ptr(), db.data_ptr() if bias else None, ws.data_ptr() if size else None, size,
            xt, wt)
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
        x, mean, rstd, weight = ctx.saved_tensors
        dx, dw, db = layer_norm_bwd(dy, x, mean, rstd, weight, ctx.bias)
        return dx, dw, db, None


def layer_norm(x, weight, bias=None, eps=1e-5):
    """Differentiable layer norm over the last axis (see ``layer_norm_fwd``)."""
    _no_capture("layer_norm", x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, eps)


# ---------------------------------------------------------------------------------------------- differential attention
def _aligned(t):
    """t, or a copy of it where its rows cannot be read 16 bytes at a time (its strides, in elements, with it); an axis of one
    element has no stride that matters."""
    st = t.stride()
    if not t.data_ptr() % 16 and t.is_contiguous() and not (st[0] | st[1] | st[2]) % 8 and st[1] < 1 << 24:
        return t, st[:-1]
    st = [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
    if t.numel() and (t.data_ptr() % 16 or t.stride(-1) != 1 or any(s % 8 or s >= 1 << 24 for s in st[1:-1]) or st[0] % 8 or
                      st[2] * t.shape[2] >= 1 << 29):
        t = t.clone(memory_format=torch.contiguous_format)
        st = [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
    return t, st[:-1]


def _lens(name, lens, b, dev):
    if lens is None:
        return None
    if lens.dtype != torch.int32 or tuple(lens.shape) != (b,) or lens.device != dev:
        raise ValueError(f"{name}: {b} int32 lengths on {dev}, got {tuple(lens.shape)} {lens.dtype} on {lens.device}")
    return lens.contiguous()


def _attn_args(name, q, k, v, lam, causal, scale, q_lens, kv_lens):
    qsh, ksh, dt = q.shape, k.shape, q.dtype
    if len(qsh) != 5 or qsh[3] != 2:
        raise ValueError(f"{name}: q of shape (B, T, H, 2, D), got {tuple(qsh)}")
    B, T, H, _, D = qsh
    if len(ksh) != 5 or ksh[0] != B or ksh[3] != 2 or ksh[4] != D:
        raise ValueError(f"{name}: k of shape ({B}, S, Hkv, 2, {D}), got {tuple(ksh)}")
    S, Hkv = ksh[1], ksh[2]
    if v.shape != (B, S, Hkv, 2 * D):
        raise ValueError(f"{name}: v of shape {(B, S, Hkv, 2 * D)}, got {tuple(v.shape)}")
    if D not in (32, 64, 128):
        raise NotImplementedError(f"{name}: maps of width 32, 64 or 128, got {D}")
    if H < 1 or Hkv < 1 or H % Hkv:
        raise ValueError(f"{name}: {H} query heads over {Hkv} key heads")
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise TypeError(f"{name}: bfloat16 or float16, got {dt}")
    if k.dtype is not dt or v.dtype is not dt:
        raise TypeError(f"{name}: q, k and v of one type, got {dt}, {k.dtype}, {v.dtype}")
    if lam.shape != (H,) or lam.dtype is not torch.float32:
        raise ValueError(f"{name}: lam of {H} float32 values, got {tuple(lam.shape)} {lam.dtype}")
    _device(name, q, k, v, lam)
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{name}: scale > 0, got {scale}")
    (q, qs), (k, ks), (v, vs), lam = _aligned(q), _aligned(k), _aligned(v), lam.contiguous()
    ql, kl = _lens(name + " q_lens", q_lens, B, q.device), _lens(name + " kv_lens", kv_lens, B, q.device)
    a = DiffAttn(q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), None, None, None, None,
                 None if ql is None else ql.data_ptr(), None if kl is None else kl.data_ptr(), *qs, *ks, *vs, scale, B, T,
                 S, H, Hkv, D, 1 if causal else 0, _TYPES[dt])
    return a, (q, k, v, lam, ql, kl)


def diff_attention_fwd(q, k, v, lam, causal=False, scale=None, q_lens=None, kv_lens=None, save=True):
    """(out, saved): out = (softmax(q1 k1^T scale) - lam softmax(q2 k2^T scale)) v, of shape (B, T, H, 2 D).

    q: (B, T, H, 2, D) -- the two maps' queries of a head side by side; k: (B, S, Hkv, 2, D); v: (B, S, Hkv, 2 D); H a
    multiple of Hkv (key head j serves the query heads j H / Hkv ...); bfloat16 or float16, D in {32, 64, 128}; lam: (H,)
    float32.  Any strides with the last axis contiguous and 16-byte aligned rows are read in place (a slice of a cache),
    others from a copy.  scale: 1 / sqrt(D) unless given.  q_lens / kv_lens: (B,) int32 device tensors, the valid
    positions and keys of each sequence, held to [0, T] / [0, S]; what stands behind them does not count.  causal: position t
    sees the keys up to t + kv_len - q_len, so one new token (T = 1) sees its whole cache.  Rows that see no key, and
    positions behind q_lens, are zeros.  A probability is held to two 16-bit terms (2^-16 of itself, float16 2^-22, there at least
    2^-39 of its row's largest).  ``saved`` is for ``diff_attention_bwd`` (None with ``save=False``)."""
    a, keep = _attn_args("diff_attention", q, k, v, lam, causal, scale, q_lens, kv_lens)
    out = q.new_empty((a.B, a.T, a.H, 2 * a.D))
    saved = None
    a.o = out.data_ptr()
    if save:
        parts = q.new_empty((3, a.B, a.T, a.H, 2 * a.D))     # the second map's and its remainder, out's remainder
        stat = q.new_empty((2, a.B * a.H * a.T), dtype=torch.float32)
        a.o2, a.ol, a.stat = parts.data_ptr(), parts.data_ptr() + 4 * out.numel(), stat.data_ptr()
        saved = (parts, stat)
    if out.numel():
        ref = C.byref(a)
        size = query("ctr_diffattn_fwd_ws_size", ref)
        ws = q.new_empty(size, dtype=torch.uint8) if size else None
        _launch(q, "ctr_diffattn_fwd", ref, ws.data_ptr() if size else None, size)
    return out, saved


def diff_attention_bwd(dout, q, k, v, lam, out, saved, causal=False, scale=None, q_lens=None, kv_lens=None):
    """(dq, dk, dv, dlam) of ``diff_attention_fwd``, given its out and saved and the same other arguments.  dS and P_1 - lam P_2 are
    rounded once to the inputs' type, in float16 held to at least 2^-36 of the row's (dq) or key's (dk, dv) largest."""
    a, keep = _attn_args("diff_attention_bwd", q, k, v, lam, causal, scale, q_lens, kv_lens)
    shape = (a.B, a.T, a.H, 2 * a.D)
    if saved is None:
        raise ValueError("diff_attention_bwd: the forward ran with save=False")
    parts, stat = saved
    for t, what in ((dout, "dout"), (out, "out")):
        if tuple(t.shape) != shape or t.dtype != q.dtype:
            raise ValueError(f"diff_attention_bwd: {what} of shape {shape} {q.dtype}, got {tuple(t.shape)} {t.dtype}")
    if tuple(parts.shape) != (3, *shape) or parts.dtype != q.dtype or not parts.is_contiguous() or \
            tuple(stat.shape) != (2, a.B * a.H * a.T) or stat.dtype != torch.float32 or not stat.is_contiguous():
        raise ValueError("diff_attention_bwd: saved as diff_attention_fwd gave it")
    _device("diff_attention_bwd", q, dout, out, parts, stat)
    (dout, gs), (out, _) = _aligned(dout), _aligned(out.contiguous())
    dq, dk, dv, dlam = q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(v.shape), lam.new_empty(a.H)
    a.o, a.stat = out.data_ptr(), stat.data_ptr()
    a.o2, a.ol = parts.data_ptr(), parts.data_ptr() + 4 * out.numel()
    ref = C.byref(a)
    size = query("ctr_diffattn_bwd_ws_size", ref)
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _launch(q, "ctr_diffattn_bwd", ref, dout.data_ptr(), *gs, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            dlam.data_ptr(), ws.data_ptr() if size else None, size)
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
        q, k, v, lam, out, q_lens, kv_lens, *saved = ctx.saved_tensors
        grads = diff_attention_bwd(dout, q, k, v, lam, out, tuple(saved), *ctx.args, q_lens, kv_lens)
        return (*grads, None, None, None, None)


def diff_attention(q, k, v, lam, causal=False, scale=None, q_lens=None, kv_lens=None):
    """Differentiable differential attention (see ``diff_attention_fwd``)."""
    _no_capture("diff_attention", q, k, v, lam)
    return _DiffAttention.apply(q, k, v, lam, causal, scale, q_lens, kv_lens)


# ---------------------------------------------------------------------------------------------- Newton-Schulz
@torch.no_grad()
def newton_schulz(mats, steps=5, coeffs=NS_COEFFS, eps=1e-7):
    """Orthogonalised matrices: X = G / (||G||_F + eps), then ``steps`` times X <- (a I + b A + c A^2) X with A = X X^T (of
    the transpose when G has more rows than columns).  mats: a matrix, a batch (..., m, n) or a list of matrices of any
    shapes (sides up to 65536) and one type (float32, bfloat16, float16); the result likewise.  Computed to float32's accuracy in the norm
    whatever the type (an element is held to 2^-22 of itself or 2^-37 of the norm, whichever is more).  Coefficients
    under which a singular value could leave [0, 7.5] are refused."""
    single = isinstance(mats, torch.Tensor)
    lst = [mats] if single else list(mats)
    if not lst:
        return []
    dt, idx = lst[0].dtype, lst[0].get_device()
    odd = [t.dtype for t in lst if t.dtype is not dt or dt not in _TYPES]
    if odd:
        raise TypeError(f"newton_schulz: one of float32, bfloat16, float16 for all, got {odd[0]}")
    out, keep, words = [], [], []
    for t in lst:
        shape = t.shape
        if len(shape) != 2 and (len(shape) < 2 or not single):
            raise ValueError(f"newton_schulz: matrices, got a shape of {tuple(shape)}")
        if t.get_device() != idx or idx < 0:
            raise ValueError(f"newton_schulz: device tensors of one device, got {t.device}")
        m, n = shape[-2:]
        o = torch.empty_like(t, memory_format=torch.contiguous_format)
        out.append(o)
        if not t.is_contiguous() and (len(shape) > 2 or (t.stride(1) != 1 and n > 1) or (t.stride(0) < n and m > 1)):
            t = t.contiguous()
            keep.append(t)          # until the launch
        src, dst, step = t.data_ptr(), o.data_ptr(), m * n * t.element_size()
        ld = n if t.is_contiguous() else max(t.stride(0), n)
        for b in range(t.numel() // (m * n) if m and n else 0):
            words += (src + b * step, dst + b * step, ld, n, n << 32 | m)
    if not 1 <= int(steps) <= 64:
        raise ValueError(f"newton_schulz: steps in [1, 64], got {steps}")
    count = len(words) // 5
    if count:
        arr = (NsMat * count).from_buffer(array.array("Q", words))
        a, b, c = coeffs
        size = query("ctr_newton_schulz_ws_size", arr, count)
        ws = out[0].new_empty(size, dtype=torch.uint8) if size else None
        _launch(out[0], "ctr_newton_schulz", arr, count, int(steps), a, b, c, eps, _TYPES[dt],
                ws.data_ptr() if size else None, size)
    return out[0] if single else out
