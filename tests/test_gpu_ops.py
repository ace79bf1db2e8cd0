"""Layer norm, differential attention and Newton-Schulz (tossctr.ops) on the GPU against their definitions in 64 bits.

Tolerances.  u = eps / 2 of the rows' type (bf16 2^-8, fp16 2^-11, fp32 2^-24) is the most a rounding changes a value,
relative to it.  The attention's bounds are per element: every rounding to 16 bits that the kernels make (P and dS as matrix
operands, o2 and out that the row sums of the backward are taken from, the results) is carried to the output by the
triangle inequality with the reference's own absolute values; fp32 work under it (scores of up to 128 products, exp2,
sums of up to 2^13 terms in lanes and trees) is held to 2^-14 of the same absolute sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
EPS32 = 2.0 ** -14
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def rel(a, b):
    return float((a.double() - b).norm() / (b.norm() + 1e-300))


# ---------------------------------------------------------------------------------------------- layer norm
def ln_ref(x, w, b, dy, eps):
    x, w = x.double().requires_grad_(), w.double().requires_grad_()
    b = b.double().requires_grad_() if b is not None else None
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    y = xc / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps) * w + (b if b is not None else 0.0)
    grads = torch.autograd.grad(y, [x, w] + ([b] if b is not None else []), dy.double())
    return y.detach(), grads


# norm-wise: a result's rounding is u; in fp32 a statistic takes at most 8 serial and log2(N / 8) tree roundings, a weight
# gradient as many as a block has rows; with means of at most two deviations 2^-17 = 128 steps of 2^-24 covers them
def ln_tol(dt):
    return U[dt] + 2.0 ** -17


@pytest.mark.parametrize("m,n,xt,wt,bias", [
    (1, 1, F32, F32, True), (3, 7, BF, F32, True), (64, 32, BF, BF, True), (257, 33, HF, F32, False),
    (130, 100, F32, F32, True), (65, 256, BF, F32, True), (33, 500, HF, HF, True), (70, 1001, BF, F32, True),
    (19, 2048, HF, F32, False), (9, 4097, BF, F32, True), (7, 8192, F32, F32, True), (5, 16381, BF, F32, True),
    (3, 20003, HF, F32, True), (5000, 64, BF, F32, True), (1, 4096, BF, F32, True), (3001, 17, F32, F32, True)])
def test_layer_norm(m, n, xt, wt, bias):
    import tossctr
    g = gen(m * 131 + n)
    x, dy = (randn(g, m, n) + randn(g, m, 1)).to(xt), randn(g, m, n).to(xt)
    w, b = (1 + 0.2 * randn(g, n)).to(wt), randn(g, n).to(wt) if bias else None
    ref, grads = ln_ref(x, w, b, dy, 1e-5)
    y, mean, rstd = tossctr.layer_norm_fwd(x, w, b, 1e-5)
    out = tossctr.layer_norm_bwd(dy, x, mean, rstd, w, bias)
    assert y.dtype == xt and out[0].dtype == xt and out[1].dtype == wt
    assert rel(y, ref) <= ln_tol(xt)
    # dx is a difference of terms of dy's size: with one element it is zero, so it is held to dy w rstd
    size = (dy.double() * w.double() * rstd.double()[:, None]).norm()
    assert float((out[0].double() - grads[0]).norm()) <= ln_tol(xt) * float(grads[0].norm() + size)
    # xhat = (x - mean) rstd is off by e |xhat| from rstd and by e rstd avg|x| <= e (rstd |mean| + 1) from the mean, which
    # counts alone where x is near the mean (avg|x| <= |mean| + the deviation, and rstd times that is at most 1)
    off, rs = mean.double()[:, None], rstd.double()[:, None]
    spread = (dy.double().abs() * (((x.double() - off) * rs).abs() + rs * off.abs() + 1)).sum(0)
    assert bool(((out[1].double() - grads[1]).abs() <= U[wt] * grads[1].abs() + 2.0 ** -17 * spread + 1e-30).all())
    if bias:
        assert bool(((out[2].double() - grads[2]).abs()
                     <= U[wt] * grads[2].abs() + 2.0 ** -17 * dy.double().abs().sum(0)).all())
    else:
        assert out[2] is None
    again = tossctr.layer_norm_bwd(dy, x, mean, rstd, w, bias)
    assert all(torch.equal(a, b) for a, b in zip(out, again) if a is not None)


def test_layer_norm_strides_and_shapes():
    import tossctr
    g = gen(5)
    big = randn(g, 6, 9, 200).to(BF)
    w, b = 1 + 0.2 * randn(g, 101), randn(g, 101)
    for x in (big[:, :, 3:104], big[:, 2:5, 3:104], big[1, ::2, 40:141], big[2, 3, :101],
              big.transpose(0, 1)[:, :, 5:106], big[:1, :1, :101].expand(4, 3, 101)):
        dy = randn(g, *x.shape).to(BF)
        y, mean, rstd = tossctr.layer_norm_fwd(x, w, b)
        dx, dw, db = tossctr.layer_norm_bwd(dy, x, mean, rstd, w)
        xc, dyc = x.contiguous(), dy.contiguous()
        y2, m2, r2 = tossctr.layer_norm_fwd(xc, w, b)
        ref = tossctr.layer_norm_bwd(dyc, xc, m2, r2, w)
        assert y.shape == x.shape and torch.equal(y, y2)
        assert torch.equal(dx, ref[0]) and torch.equal(dw, ref[1]) and torch.equal(db, ref[2])


def test_layer_norm_empty_rows_and_offset():
    import tossctr
    w, b = torch.ones(40, device="cuda"), torch.zeros(40, device="cuda")
    x = torch.empty(0, 40, device="cuda", dtype=BF)
    y, mean, rstd = tossctr.layer_norm_fwd(x, w, b)
    dx, dw, db = tossctr.layer_norm_bwd(x, x, mean, rstd, w)
    assert y.shape == (0, 40) and dx.shape == (0, 40) and not dw.any() and not db.any()
    # a mean of 1000 deviations: its fp32 rounding is 1000 2^-24 of a deviation, no more
    g = gen(6)
    x = randn(g, 50, 700) + 1000
    y, _, _ = tossctr.layer_norm_fwd(x, torch.ones(700, device="cuda"), None)
    ref, _ = ln_ref(x, torch.ones(700, device="cuda"), None, x, 1e-5)
    assert rel(y, ref) <= 16 * 1000 * 2.0 ** -24


def test_layer_norm_autograd_and_differences():
    import tossctr
    g = gen(7)
    x, w, b = randn(g, 6, 20), 1 + 0.2 * randn(g, 20), randn(g, 20)
    dy = randn(g, 6, 20)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    tossctr.layer_norm(*leaves).backward(dy)
    h = 2.0 ** -6
    for k, leaf in enumerate(leaves):
        d = randn(g, *leaf.shape)
        ends = []
        for s in (h, -h):
            args = [x, w, b]
            args[k] = args[k] + s * d
            ends.append(float((tossctr.layer_norm_fwd(*args)[0].double() * dy.double()).sum()))
        num, ana = (ends[0] - ends[1]) / (2 * h), float((leaf.grad.double() * d.double()).sum())
        # central differences: h^2 times a third derivative of order |d|^3, and the two values' fp32 noise over 2 h
        scale = float(dy.norm() * d.norm())
        assert abs(num - ana) <= scale * (h * h * float(d.norm()) ** 2 + 2.0 ** -20 / h)


# ---------------------------------------------------------------------------------------------- differential attention
def da_ref(q, k, v, lam, do, causal, scale, q_lens, kv_lens):
    """The definition in 64 bits, its gradients, and the bounds of the kernels' roundings."""
    u = U[q.dtype]
    B, T, H, _, D = q.shape
    S, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    dev = q.device
    ql = q_lens.long().clamp(0, T) if q_lens is not None else torch.full((B,), T, device=dev)
    kl = kv_lens.long().clamp(0, S) if kv_lens is not None else torch.full((B,), S, device=dev)
    i, j = torch.arange(T, device=dev), torch.arange(S, device=dev)
    seen = (j[None, None] < kl[:, None, None]) & (i[None, :, None] < ql[:, None, None])
    if causal:
        seen = seen & (j[None, None] <= i[None, :, None] + (kl - ql)[:, None, None])
    seen = seen[:, None]
    behind = (j[None] >= kl[:, None])
    kd = k.double().masked_fill(behind[:, :, None, None, None], 0.0)
    vd = v.double().masked_fill(behind[:, :, None, None], 0.0)
    late = (i[None] >= ql[:, None])
    qd = q.double().masked_fill(late[:, :, None, None, None], 0.0)
    kk = kd.repeat_interleave(G, 2).permute(3, 0, 2, 1, 4)          # 2 B H S D
    vv = vd.repeat_interleave(G, 2).transpose(1, 2)                 # B H S DV
    qq = qd.permute(3, 0, 2, 1, 4)                                  # 2 B H T D
    s = (qq @ kk.transpose(-1, -2)) * scale
    # a score's fp32 value, its product with log2(e) and the difference to the maximum are each off by half a step of
    # the largest score, and that is the exponential's relative error
    EPS32 = 2.0 ** -14 + 3 * 2.0 ** -24 * 1.4427 * float(s.abs().max()) if s.numel() else 0.0
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    tot = p.sum(-1, keepdim=True)
    p = p / torch.where(tot == 0, 1.0, tot)
    lm = lam.double()[None, :, None, None]
    o = p @ vv
    out = o[0] - lm * o[1]
    pv = p @ vv.abs()
    # P's rounding, and the result's
    b_out = u * out.abs() + (u + EPS32) * (pv[0] + lm.abs() * pv[1])
    res = {"out": (out.transpose(1, 2), b_out.transpose(1, 2))}
    if do is None:
        return res
    dd = do.double().masked_fill(late[:, :, None, None], 0.0).transpose(1, 2)       # B H T DV
    dp = dd @ vv.transpose(-1, -2)
    d1, d2 = (dd * o[0]).sum(-1, keepdim=True), (dd * o[1]).sum(-1, keepdim=True)
    ds = torch.stack([p[0] * (dp - d1), -lm * p[1] * (dp - d2)])
    adp = dd.abs() @ vv.abs().transpose(-1, -2)
    # the row sums are taken from out and o2 as they were rounded
    e2 = (dd.abs() * (u * o[1].abs() + (u + EPS32) * pv[1])).sum(-1, keepdim=True)
    e1 = (dd.abs() * b_out.transpose(1, 2).transpose(1, 2)).sum(-1, keepdim=True) + lm.abs() * e2
    eds = torch.stack([u * ds[0].abs() + p[0] * (e1 + EPS32 * (adp + (dd * o[0]).abs().sum(-1, keepdim=True))),
                       u * ds[1].abs() + lm.abs() * p[1] * (e2 + EPS32 * (adp + (dd * o[1]).abs().sum(-1, keepdim=True)))])
    ads = ds.abs()

    def heads(t):        # sum over the query heads of a key head
        return t.unflatten(-3, (Hkv, G)).sum(-3)

    dq = scale * (ds @ kk)
    b_dq = u * dq.abs() + scale * ((eds + EPS32 * ads) @ kk.abs())
    dk = scale * heads(ds.transpose(-1, -2) @ qq)
    b_dk = u * dk.abs() + scale * heads((eds + EPS32 * ads).transpose(-1, -2) @ qq.abs())
    pc = p[0] - lm * p[1]
    dv = heads(pc.transpose(-1, -2) @ dd)
    b_dv = u * dv.abs() + heads((u * pc.abs() + EPS32 * (p[0] + lm.abs() * p[1])).transpose(-1, -2) @ dd.abs())
    res["dq"] = tuple(t.permute(1, 3, 2, 0, 4) for t in (dq, b_dq))
    res["dk"] = tuple(t.permute(1, 3, 2, 0, 4) for t in (dk, b_dk))
    res["dv"] = tuple(t.transpose(1, 2) for t in (dv, b_dv))
    res["dlam"] = (-d2.sum((0, 2, 3)), EPS32 * (p[1] * adp).sum((0, 2, 3)))      # in fp32 throughout: no 16-bit rounding
    return res


# results below fp16's smallest step are rounded to it; a probability below fp32's smallest normal number, 2^-126, comes out 0,
# and what it would have multiplied (a gradient's dP, a query, over all rows: below 2^26 here) stays under 2^-100
TINY = {BF: 2.0 ** -100, HF: 2.0 ** -24}


def hold(name, got, ref, bound, dt):
    over = (got.double() - ref).abs() - bound - (TINY[dt] if got.dtype == dt else 0.0)
    assert bool((over <= 0).all()), (name, float(over.max()), float(bound.max()))


def da_inputs(g, B, T, S, H, Hkv, D, dt):
    return (randn(g, B, T, H, 2, D).to(dt), randn(g, B, S, Hkv, 2, D).to(dt), randn(g, B, S, Hkv, 2 * D).to(dt),
            0.8 * torch.rand(H, device="cuda", generator=g) - 0.1, randn(g, B, T, H, 2 * D).to(dt))


def da_case(q, k, v, lam, do, causal=False, scale=None, q_lens=None, kv_lens=None):
    import tossctr
    kw = dict(causal=causal, scale=scale, q_lens=q_lens, kv_lens=kv_lens)
    sc = scale if scale is not None else 1 / math.sqrt(q.shape[-1])
    ref = da_ref(q, k, v, lam, do, causal, sc, q_lens, kv_lens)
    out, saved = tossctr.diff_attention_fwd(q, k, v, lam, **kw)
    hold("out", out, *ref["out"], q.dtype)
    light, none = tossctr.diff_attention_fwd(q, k, v, lam, save=False, **kw)
    assert none is None and torch.equal(light, out)
    grads = tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved, **kw)
    for name, got in zip(("dq", "dk", "dv", "dlam"), grads):
        hold(name, got, *ref[name], q.dtype)
    again = tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved, **kw)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    return out, grads


@pytest.mark.parametrize("B,T,S,H,Hkv,D,dt,causal", [
    (1, 1, 1, 1, 1, 32, BF, False), (2, 1, 77, 4, 2, 64, BF, True), (3, 5, 5, 3, 1, 32, HF, True),
    (2, 33, 65, 6, 2, 64, HF, False), (2, 60, 60, 4, 4, 32, BF, False), (1, 129, 300, 8, 1, 128, BF, True),
    (2, 100, 31, 2, 2, 128, HF, True), (1, 513, 513, 4, 2, 64, BF, True), (1, 7, 2049, 5, 5, 128, BF, False),
    (4, 1, 4000, 8, 1, 32, BF, False), (1, 1, 9001, 6, 2, 128, HF, False), (30, 140, 140, 9, 9, 32, BF, True),
    (20, 260, 97, 16, 8, 64, HF, False), (1, 257, 1100, 64, 64, 128, BF, True)])
def test_diff_attention(B, T, S, H, Hkv, D, dt, causal):
    da_case(*da_inputs(gen(B * 1000 + T + S + D), B, T, S, H, Hkv, D, dt), causal=causal)


@pytest.mark.parametrize("dt,D,causal", [(BF, 64, True), (HF, 32, False), (BF, 128, True)])
def test_diff_attention_lengths(dt, D, causal):
    """Sequences of no key, one key, ends inside a tile, fewer keys than positions, lengths past the tensor; what stands
    behind the ends is NaN."""
    B, T, S, H, Hkv = 8, 70, 150, 4, 2
    q, k, v, lam, do = da_inputs(gen(11 + D), B, T, S, H, Hkv, D, dt)
    kv = torch.tensor([0, 1, 150, 37, 64, 40, 1000, 150], device="cuda", dtype=torch.int32)
    ql = torch.tensor([70, 70, 0, 1, 64, 70, 70, -3], device="cuda", dtype=torch.int32)
    for b in range(B):
        k[b, max(0, min(S, int(kv[b]))):] = math.nan
        v[b, max(0, min(S, int(kv[b]))):] = math.nan
        q[b, max(0, min(T, int(ql[b]))):] = math.nan
    out, (dq, dk, dv, _) = da_case(q, k, v, lam, do, causal=causal, q_lens=ql, kv_lens=kv)
    assert not out[0].any() and not out[2].any() and not dk[1, 1:].any() and not dv[7].any() and not dq[3, 1:].any()


@pytest.mark.parametrize("dt,G,D", [(BF, 1, 64), (HF, 2, 32), (BF, 3, 128)])
def test_diff_attention_rows_that_see_nothing(dt, G, D):
    """Causal with fewer keys than positions: the first 13 positions see nothing.  NaN in their queries and gradients reaches no
    one, and NaN in the values that other rows see does not reach them."""
    import tossctr
    B, T, S, Hkv = 2, 45, 50, 2
    q, k, v, lam, do = da_inputs(gen(71 + D), B, T, S, G * Hkv, Hkv, D, dt)
    lens = torch.tensor([32, 32], device="cuda", dtype=torch.int32)
    q[:, :13] = 0.0
    do[:, :13] = 0.0
    want, want_grads = da_case(q, k, v, lam, do, causal=True, kv_lens=lens)
    q[:, :13] = math.nan
    do[:, :13] = math.nan
    out, saved = tossctr.diff_attention_fwd(q, k, v, lam, causal=True, kv_lens=lens)
    grads = tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved, causal=True, kv_lens=lens)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))
    v[:, :32] = math.nan
    out, _ = tossctr.diff_attention_fwd(q, k, v, lam, causal=True, kv_lens=lens)
    assert not out[:, :13].any() and bool(out[:, 13:].isnan().all())


def test_diff_attention_large_scores_and_signs():
    """Scores of hundreds (one key takes all), equal maps with lam = 1 (the difference is zero but for roundings), lam of
    either sign, a scale of its own."""
    q, k, v, lam, do = da_inputs(gen(21), 2, 90, 200, 4, 2, 64, BF)
    da_case(q * 16, k * 4, v, lam, do, causal=True, scale=0.25)
    q[:, :, :, 1] = q[:, :, :, 0]
    k[:, :, :, 1] = k[:, :, :, 0]
    out, _ = da_case(q, k, v, torch.ones_like(lam), do)
    da_case(q, k, v, torch.tensor([-3.0, 0.0, 2.5, 1e-3], device="cuda"), do)


@pytest.mark.parametrize("size", [1e-6, 3e4])
def test_diff_attention_fp16_gradient_sizes(size):
    """fp16 gradients of any size keep their relative accuracy: dO of 1e-6 (values under fp16's normal range are exact
    multiples of its smallest step, so dO is rounded first) and of 3e4."""
    q, k, v, lam, do = da_inputs(gen(31), 1, 200, 1500, 4, 2, 64, HF)
    da_case(q, k, v * (1 if size < 1 else 0.01), lam, (do * size).clamp(-6e4, 6e4).to(HF))


def test_diff_attention_strides():
    """A slice of a longer cache, heads and maps as they come out of one projection, an odd offset (read from a copy)."""
    import tossctr
    g = gen(41)
    B, T, S, H, D = 2, 20, 50, 4, 64
    proj = randn(g, B, T, 3 * H * 2 * D + 3).to(BF)
    cache = randn(g, B, H, 2 * S, 4 * D).to(BF)
    lam = torch.rand(H, device="cuda", generator=g)
    kc, vc = cache[:, :, 5:5 + S, :2 * D].unflatten(-1, (2, D)).transpose(1, 2), cache[:, :, 5:5 + S, 2 * D:].transpose(1, 2)
    do = randn(g, B, H, T, 2 * D).to(BF).transpose(1, 2)
    for off in (0, 3):
        q = proj[:, :, off:off + H * 2 * D].unflatten(-1, (2, H, D)).transpose(2, 3)
        kw = dict(causal=True)
        out, saved = tossctr.diff_attention_fwd(q, kc, vc, lam, **kw)
        got = tossctr.diff_attention_bwd(do, q, kc, vc, lam, out, saved, **kw)
        qc, k2, v2 = q.contiguous(), kc.contiguous(), vc.contiguous()
        out2, saved2 = tossctr.diff_attention_fwd(qc, k2, v2, lam, **kw)
        ref = tossctr.diff_attention_bwd(do.contiguous(), qc, k2, v2, lam, out2, saved2, **kw)
        assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(got, ref))


def test_diff_attention_empty():
    import tossctr
    lam = torch.rand(2, device="cuda")
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=BF)  # noqa: E731
    out, saved = tossctr.diff_attention_fwd(z(3, 4, 2, 2, 32), z(3, 0, 1, 2, 32), z(3, 0, 1, 64), lam)
    assert out.shape == (3, 4, 2, 64) and not out.any()
    dq, dk, dv, dl = tossctr.diff_attention_bwd(out, z(3, 4, 2, 2, 32), z(3, 0, 1, 2, 32), z(3, 0, 1, 64), lam, out, saved)
    assert not dq.any() and dk.shape[1] == 0 and not dl.any()
    for b, t in ((3, 0), (0, 4)):
        q, k, v = z(b, t, 2, 2, 32), z(b, 7, 1, 2, 32), z(b, 7, 1, 64)
        out, saved = tossctr.diff_attention_fwd(q, k, v, lam)
        dq, dk, dv, dl = tossctr.diff_attention_bwd(out, q, k, v, lam, out, saved)
        assert out.numel() == 0 and dq.numel() == 0 and not dk.any() and not dv.any() and not dl.any()


def test_diff_attention_autograd_matches_bwd():
    import tossctr
    q, k, v, lam, do = da_inputs(gen(51), 2, 40, 40, 4, 2, 32, BF)
    lens = torch.tensor([40, 17], device="cuda", dtype=torch.int32)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, lam)]
    tossctr.diff_attention(*leaves, causal=True, q_lens=lens, kv_lens=lens).backward(do)
    out, saved = tossctr.diff_attention_fwd(q, k, v, lam, True, None, lens, lens)
    ref = tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved, True, None, lens, lens)
    assert all(torch.equal(a.grad, b) for a, b in zip(leaves, ref))


@pytest.mark.parametrize("dt", [BF, HF])
def test_diff_attention_short_rows_keep_their_precision(dt):
    """Two roundings reach dQ and dK, of dS and of the result, of one relative size and independent: sqrt(2) of the result's own
    rounding in the norm.  A third, of the row sums, would make it sqrt(3); 1.5 stands between (1.41 < 1.5 < 1.73)."""
    import tossctr
    q, k, v, lam, do = da_inputs(gen(57), 7, 17, 17, 4, 2, 128, dt)
    ref = da_ref(q, k, v, lam, do, True, 128 ** -0.5, None, None)
    out, saved = tossctr.diff_attention_fwd(q, k, v, lam, causal=True)
    dq, dk, _, _ = tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved, causal=True)
    for name, got in (("dq", dq), ("dk", dk)):
        want = ref[name][0]
        assert float((got.double() - want).norm()) <= 1.5 * float((want.to(dt).double() - want).norm()), name


def test_diff_attention_gradient_of_a_sum():
    """The gradient that arrives is one element for all places (strides of 0)."""
    import tossctr
    q, k, v, lam, _ = da_inputs(gen(53), 2, 37, 37, 4, 2, 64, BF)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    out = tossctr.diff_attention(*leaves, causal=True)
    out.sum().backward()
    with torch.no_grad():
        o, saved = tossctr.diff_attention_fwd(q, k, v, lam, causal=True)
        want = tossctr.diff_attention_bwd(torch.ones_like(o), q, k, v, lam, o, saved, causal=True)
    for t, w in zip(leaves, want):
        assert torch.equal(t.grad, w)


def test_diff_attention_gradient_by_differences():
    """dlam and dV are exact differences (the output is linear in them); dQ and dK against central differences of the
    definition in 64 bits, through the bounds of the kernels' gradients."""
    q, k, v, lam, do = da_inputs(gen(61), 1, 9, 14, 2, 1, 32, HF)
    _, (dq, dk, dv, dlam) = da_case(q, k, v, lam, do)
    ref = da_ref(q, k, v, lam, do, False, 32 ** -0.5, None, None)

    def loss(q, k, v, lam):
        return float((da_ref(q, k, v, lam, None, False, 32 ** -0.5, None, None)["out"][0] * do.double()).sum())

    args, h = [t.double() for t in (q, k, v, lam)], 1e-4
    U[torch.float64] = 0.0
    for n, (name, got) in enumerate((("dq", dq), ("dk", dk), ("dv", dv), ("dlam", dlam))):
        d = randn(gen(70 + n), *got.shape).double()
        hi, lo = ([a + s * h * d if i == n else a for i, a in enumerate(args)] for s in (1, -1))
        num = (loss(*hi) - loss(*lo)) / (2 * h)
        bound = float((ref[name][1] * d.abs()).sum()) + 1e-6 * float(do.double().norm() * d.norm())
        assert abs(num - float((got.double() * d).sum())) <= bound, name


# ---------------------------------------------------------------------------------------------- Newton-Schulz
COEFFS = (3.4445, -4.7750, 2.0315)


def ns_ref(g, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = g.double()
    x = x if x.shape[0] <= x.shape[1] else x.t()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x if g.shape[0] <= g.shape[1] else x.t()


# four roundings of 2^-22 a step (the planes of X, A and W, and the sums) relative to ||X||, each multiplied by at most
# a = 3.4445 in every later step: 4 2^-22 (3.4445^5 - 1) / 2.4445, and the result's own
NS_TOL = 4 * 2.0 ** -22 * (3.4445 ** 5 - 1) / 2.4445


@pytest.mark.parametrize("shapes,dt", [
    ([(1, 1)], F32), ([(1, 50), (50, 1), (2, 3)], F32), ([(96, 32), (32, 32), (384, 32), (32, 384)], F32),
    ([(64, 64), (128, 128), (100, 200), (37, 11)], BF), ([(64, 448)], F32), ([(24, 976), (31, 1000)], HF),
    ([(129, 130)], F32), ([(256, 300), (700, 129), (5, 2000), (3000, 40)], F32), ([(513, 1025)], BF),
    ([(1000, 384)], HF), ([(40, 40)] * 23 + [(150, 200)] * 21, F32)])
def test_newton_schulz(shapes, dt):
    import tossctr
    g = gen(len(shapes) * 7 + shapes[0][0])
    mats = [(randn(g, m, n) * 1e-3).to(dt) for m, n in shapes]
    out = tossctr.newton_schulz(mats)
    for m, o in zip(mats, out):
        assert o.dtype == dt and o.shape == m.shape
        assert rel(o, ns_ref(m)) <= U[dt] + NS_TOL, tuple(m.shape)
    assert all(torch.equal(a, b) for a, b in zip(out, tossctr.newton_schulz(mats)))


@pytest.mark.parametrize("shapes,dt", [([(801, 900), (1100, 770)], F32), ([(790, 12161)], F32), ([(12200, 771), (33, 70)], BF)])
def test_newton_schulz_large_tiles(shapes, dt):
    test_newton_schulz(shapes, dt)


def test_newton_schulz_forms():
    """Batches, strides, transposes, one step, other coefficients, zeros, sizes of 1e30 and 1e-30."""
    import tossctr
    g = gen(81)
    batch = randn(g, 3, 2, 40, 72)
    out = tossctr.newton_schulz(batch)
    assert out.shape == batch.shape
    assert all(rel(out[i, j], ns_ref(batch[i, j])) <= NS_TOL for i in range(3) for j in range(2))
    big = randn(g, 300, 400)
    for x in (big[:, 10:170], big[::2, ::2], big.t(), big[5:6], big[:, 7:8], big[20:60, 1:33]):
        assert rel(tossctr.newton_schulz(x), ns_ref(x)) <= NS_TOL
    assert rel(tossctr.newton_schulz(big, steps=1, coeffs=(1.5, -0.5, 0.0)), ns_ref(big, 1, (1.5, -0.5, 0.0))) <= NS_TOL
    assert rel(tossctr.newton_schulz(big, steps=9, coeffs=(2.0, -1.5, 0.5)), ns_ref(big, 9, (2.0, -1.5, 0.5))) <= NS_TOL
    for shape in ((40, 50), (200, 300)):
        z = torch.zeros(shape, device="cuda")
        assert not tossctr.newton_schulz(z).any()
        x = randn(g, *shape)
        for s in (1e30, 1e-30):
            assert rel(tossctr.newton_schulz(x * s, eps=0.0), ns_ref(x, eps=0.0)) <= NS_TOL
    assert tossctr.newton_schulz([]) == [] and tossctr.newton_schulz(big[:0]).shape == (0, 400)


# ---------------------------------------------------------------------------------------------- together
def test_ops_on_a_side_stream_and_in_graphs():
    """A block's norm, attention, backward passes and the update's direction, captured twice and replayed in turn with
    eager work between: every replay gives the eager bits, on new inputs too."""
    import tossctr
    g = gen(91)
    B, T, H, D = 2, 48, 4, 32
    w, b, lam = 1 + 0.1 * randn(g, 2 * D), 0.1 * randn(g, 2 * D), torch.rand(H, device="cuda", generator=g)

    def block(q, k, v, do, mats):
        out, saved = tossctr.diff_attention_fwd(q, k, v, lam, causal=True)
        y, mean, rstd = tossctr.layer_norm_fwd(out, w, b)
        dout, dw, db = tossctr.layer_norm_bwd(do, out, mean, rstd, w)
        grads = tossctr.diff_attention_bwd(dout, q, k, v, lam, out, saved, causal=True)
        return [y, dw, db, *grads, *tossctr.newton_schulz(mats)]

    def inputs(seed, S):
        gg = gen(seed)
        q, k, v, _, do = da_inputs(gg, B, T, S, H, 2, D, BF)
        return [q, k, v, do, [randn(gg, 64, 96), randn(gg, 140, 200)]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    sets = [inputs(1, 48), inputs(2, 700)]
    graphs = []
    with torch.cuda.stream(side):
        for s in sets:
            block(*s)
            eager = block(*s)
        side.synchronize()
        for s in sets:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                res = block(*s)
            graphs.append((gr, res))
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(3):
        for n, (gr, res) in enumerate(graphs):
            fresh = inputs(100 + 10 * turn + n, 48 if n == 0 else 700)
            for a, c in zip(sets[n][:4], fresh[:4]):
                a.copy_(c)
            for a, c in zip(sets[n][4], fresh[4]):
                a.copy_(c)
            want = block(*sets[n])
            gr.replay()
            graphs[1 - n][0].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(res, want))


def test_differentiable_calls_refuse_capture(monkeypatch):
    """The capture is only claimed: what has to be seen is that nothing is launched and no graph node made."""
    import tossctr
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    x, w = torch.randn(4, 32, device="cuda", requires_grad=True), torch.ones(32, device="cuda")
    with pytest.raises(RuntimeError, match="layer_norm_bwd"):
        tossctr.layer_norm(x, w)
    q, k, v, lam, _ = da_inputs(gen(1), 1, 4, 4, 1, 1, 32, BF)
    with pytest.raises(RuntimeError, match="diff_attention_bwd"):
        tossctr.diff_attention(q, k, v, lam.requires_grad_())
    with torch.no_grad():
        assert tossctr.layer_norm(x, w).shape == x.shape
    assert tossctr.layer_norm(x.detach(), w).shape == x.shape
