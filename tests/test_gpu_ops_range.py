"""Differential attention and Newton-Schulz over the range of their types (tossctr.ops): probabilities far below a row's largest,
gradients and rows of far sizes, weights of any size, structured matrices, lengths together with split keys and split rows.  Against
the definitions in 64 bits, with bounds from the roundings."""
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_ops import BF, F32, HF, NS_TOL, U, da_case, da_inputs, da_ref, gen, hold, ns_ref, randn, rel  # noqa: E402


# ---------------------------------------------------------------------------------------------- forward
def fwd_ref(q, k, v, lam, scale):
    """The output in 64 bits (no mask) and its bound: the result's own rounding u |O|; of P the two 16-bit terms leave u^2 of it,
    in float16 at least 2^-39 of the row's largest; and the fp32 steps under it -- 2 D roundings of a score's absolute sum and
    three of its value, through the exponential, and 2 S + 8 of sums, quotient and difference."""
    u, (B, T, H, _, D), S = U[q.dtype], q.shape, k.shape[1]
    G = H // k.shape[2]
    qq = q.double().permute(3, 0, 2, 1, 4)                                    # 2 B H T D
    kk = k.double().repeat_interleave(G, 2).permute(3, 0, 2, 1, 4)            # 2 B H S D
    vv = v.double().repeat_interleave(G, 2).transpose(1, 2)                   # B H S DV
    s = qq @ kk.transpose(-1, -2) * scale
    p = s.softmax(-1)
    lm = lam.double()[None, :, None, None]
    out = (p[0] - lm * p[1]) @ vv
    size = float((qq.abs() @ kk.abs().transpose(-1, -2)).max()) * scale
    eps = 2.0 ** -23 * (1.4427 * (D * size + 3 * float(s.abs().max())) + 2 * S + 8)
    pv = (p[0] + lm.abs() * p[1]) @ vv.abs()
    least = 2.0 ** -39 * (1 + lm.abs()) * vv.abs().sum(-2, keepdim=True) if q.dtype == HF else 0.0
    bound = u * out.abs() + (u * u + eps) * pv + least
    return out.transpose(1, 2), bound.transpose(1, 2)


@pytest.mark.parametrize("nats", [5.0, 12.0, 15.0, 17.0, 17.5, 19.0])
@pytest.mark.parametrize("dt,D,S,B", [(HF, 64, 4097, 3), (BF, 64, 4097, 3), (HF, 128, 700, 1), (HF, 32, 9000, 1)])
def test_one_key_far_above_the_others(dt, D, S, B, nats):
    """A first key that takes nearly all of every row and has no value, the others `nats` below it with values of one sign: what
    they give together is the output.  (9000 keys and one batch: the keys are split.)"""
    import tossctr
    g = gen(int(10 * nats) + S)
    T, H = 45, 2
    q, k = torch.zeros(B, T, H, 2, D, device="cuda"), torch.zeros(B, S, H, 2, D, device="cuda")
    q[..., 0] = 1.0
    k[:, 0, :, :, 0] = nats
    k[:, 1:, :, :, 1:] = 0.05 * randn(g, B, S - 1, H, 2, D - 1)       # the queries are 0 there but for a little
    q[..., 1:] = 0.05 * randn(g, B, T, H, 2, D - 1)
    v = 1 + 0.5 * torch.rand(B, S, H, 2 * D, device="cuda", generator=g)
    v[:, 0] = 0.0
    lam = torch.tensor([0.5, -0.25], device="cuda")
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    for t in (T, 1):
        out, _ = tossctr.diff_attention_fwd(q[:, :t], k, v, lam, scale=1.0, save=False)
        hold(f"out {t}", out, *fwd_ref(q[:, :t], k, v, lam, 1.0), dt)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,S,H,Hkv,D", [(1, 2, 4, 4, 32), (17, 3, 4, 2, 32), (40, 9, 2, 2, 64), (33, 33, 2, 1, 128)])
def test_maps_that_nearly_agree(dt, T, S, H, Hkv, D):
    """The second map's queries differ from the first's by a rounding or two and lam is 1: the difference is far smaller than
    either product, and is held to what two 16-bit terms of P leave (one term leaves up to 2^7 (bf16) times the bound)."""
    import tossctr
    g = gen(T + S)
    q, k, v, _, _ = da_inputs(g, 5, T, S, H, Hkv, D, dt)
    q, k = (q * 0.5).to(dt), (k * 0.5).to(dt)
    q[:, :, :, 1] = (q[:, :, :, 0].float() * (1 + 4 * U[dt] * randn(g, *q.shape[:3], D))).to(dt)
    k[:, :, :, 1] = k[:, :, :, 0]
    lam = torch.ones(H, device="cuda")
    out, _ = tossctr.diff_attention_fwd(q, k, v, lam, save=False)
    hold("out", out, *fwd_ref(q, k, v, lam, D ** -0.5), dt)


@pytest.mark.parametrize("D,T,S", [(64, 90, 200), (32, 3, 4000), (128, 40, 333)])
def test_large_scores_in_float16(D, T, S):
    """Scores of hundreds, one key takes all; equal maps; lam of either sign."""
    q, k, v, lam, do = da_inputs(gen(23 + D), 2, T, S, 4, 2, D, HF)
    da_case((q * 16).to(HF), (k * 4).to(HF), v, lam, do, causal=True, scale=0.25)
    q[:, :, :, 1], k[:, :, :, 1] = q[:, :, :, 0], k[:, :, :, 0]
    da_case(q, k, v, torch.ones_like(lam), do)


# ---------------------------------------------------------------------------------------------- backward
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("T,S", [(1, 1), (40, 40), (5, 300)])
def test_lam_of_any_size(dt, T, S):
    """Rows that see one key have P_1 = P_2 = 1, and P_1 - lam P_2 passes every 16-bit range that is not fitted to it."""
    q, k, v, _, do = da_inputs(gen(T + S), 2, T, S, 6, 2, 32, dt)
    lam = torch.tensor([70.0, -70.0, 1e3, -3e4, 1e-5, 0.0], device="cuda")
    da_case(q, k, (v * 2.0 ** -10).to(dt), lam, (do * 2.0 ** -6).to(dt), causal=T == S)


def floors(q, k, v, lam, do, scale):
    """What float16 leaves of dS and P_1 - lam P_2 beside u of them (no mask, one key head): scaled so that a row's (in dQ) or a
    key's (in dK, dV) largest stands at 2^11 or more, a value is held to half of the type's smallest step, 2^-25, which is 2^-36 of
    that largest; it meets every key (query, dO)."""
    qq, kk, vv, dd = (t.double().transpose(1, 2) for t in (q.flatten(3), k.flatten(3), v, do))       # B H T 2D, B 1 S 2D, ...
    D, lm = q.shape[-1], lam.double()[None, :, None, None]
    qs, ks = (qq[..., :D], qq[..., D:]), (kk[..., :D], kk[..., D:])
    p = [(a @ b.transpose(-1, -2) * scale).softmax(-1) for a, b in zip(qs, ks)]
    dp = dd @ vv.transpose(-1, -2)
    ds = [x * (dp - (x * dp).sum(-1, keepdim=True)) for x in p]
    row = 2.0 ** -36 * torch.maximum(ds[0].abs(), ds[1].abs()).amax(-1, keepdim=True)
    dq = torch.cat([scale * row * w * b.abs().sum(-2, keepdim=True) for w, b in zip((1, lm.abs()), ks)], -1)
    key = 2.0 ** -36 * torch.maximum(ds[0].abs(), (lm * ds[1]).abs()).amax((1, 2))[:, None, :, None]
    dk = torch.cat([scale * key * a.abs().sum((1, 2), keepdim=True) for a in qs], -1)
    dv = 2.0 ** -36 * (p[0] - lm * p[1]).abs().amax((1, 2))[:, None, :, None] * dd.abs().sum((1, 2), keepdim=True)
    return {"dq": dq.transpose(1, 2).unflatten(-1, (2, D)), "dk": dk.transpose(1, 2).unflatten(-1, (2, D)), "dv": dv.transpose(1, 2)}


@pytest.mark.parametrize("bits", [20, 26, 30])
def test_float16_gradients_of_keys_far_below(bits):
    """Keys whose probabilities are 2^-20 ... 2^-30 of their neighbours' in every row: their dK and dV keep their bits."""
    import tossctr
    q, k, v, lam, do = da_inputs(gen(bits), 1, 200, 64, 2, 1, 32, HF)
    q, k = 0.1 * q.float(), 0.1 * k.float()
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[:, ::2, :, :, 0] = -bits * math.log(2)
    q, k, do = q.to(HF), k.to(HF), do * 2.0 ** 10
    ref, least = da_ref(q, k, v, lam, do, False, 1.0, None, None), floors(q, k, v, lam, do, 1.0)
    out, saved = tossctr.diff_attention_fwd(q, k, v, lam, scale=1.0)
    grads = tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved, scale=1.0)
    for name, got in zip(("dq", "dk", "dv"), grads):
        hold(name, got, ref[name][0], ref[name][1] + least[name], HF)


def test_float16_rows_of_far_sizes():
    """Rows of a tile whose dS lie 2^34 apart, over keys of sizes that bring their dQ into float16's range: each keeps its bits."""
    import tossctr
    q, k, v, lam, do = da_inputs(gen(3), 2, 64, 50, 2, 2, 64, HF)
    q = (q * 2.0 ** -8).to(HF)
    q[:, ::2, ..., 0], q[:, 1::2, ..., 0] = 8.0, -8.0          # even rows see the first keys, odd ones the others
    k[:, :25] *= 2.0 ** -6
    k[:, 25:] *= 2.0 ** 5
    k[:, :25, ..., 0], k[:, 25:, ..., 0] = 8.0, -8.0
    do = do.clamp(-3, 3)
    do[:, ::2] *= 2.0 ** 14
    do[:, 1::2] = torch.sign(do[:, 1::2]) * 2.0 ** -20
    ref = da_ref(q, k, v, lam, do, False, 1.0, None, None)
    out, saved = tossctr.diff_attention_fwd(q, k, v, lam, scale=1.0)
    grads = tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved, scale=1.0)
    for name, got in zip(("dq", "dk", "dv"), grads):
        want, bound = ref[name]
        far = want.abs() >= 65520          # float16 rounds these to infinity (some of dK: 32 rows of 2^13 times 8)
        assert name == "dk" or not far.any()
        assert torch.equal(got[far].double(), torch.sign(want[far]) * math.inf)
        hold(name, got.masked_fill(far, 0.0), want.masked_fill(far, 0.0), bound.masked_fill(far, 0.0), HF)


def test_an_infinite_row_stays_alone():
    """A row whose gradient holds an infinity leaves the other rows' dQ as they are without it."""
    import tossctr
    for dt in (HF, BF):
        q, k, v, lam, do = da_inputs(gen(9), 1, 40, 70, 2, 1, 64, dt)
        got = []
        for x in (0.0, math.inf):
            do[:, 7] = 0.0
            do[:, 7, :, 3] = x
            out, saved = tossctr.diff_attention_fwd(q, k, v, lam)
            got.append(tossctr.diff_attention_bwd(do, q, k, v, lam, out, saved)[0])
        others = torch.arange(40, device="cuda") != 7
        assert torch.equal(got[0][:, others], got[1][:, others]), dt


def test_float16_small_values_keep_the_row_sums():
    """Values of a few of float16's smallest steps under gradients of thousands: the row sums of the backward come from outputs
    that a 16-bit number, and what its rounding left out at the same scale, would not hold."""
    g = gen(13)
    q, k, v, lam, do = da_inputs(g, 2, 40, 60, 4, 2, 64, HF)
    v = (v * 2.0 ** -21).to(HF)
    do = (do * 2.0 ** 13).clamp(-6e4, 6e4).to(HF)
    q, k = (q / 16).to(HF), (k * 16).to(HF)
    ref = da_ref(q, k, v, lam, do, False, 1 / 8, None, None)
    assert float(ref["dq"][0].abs().mean()) > 2.0 ** -12            # far above float16's smallest step
    da_case(q, k, v, lam, do)


# ---------------------------------------------------------------------------------------------- lengths and splits
@pytest.mark.parametrize("dt,D,T", [(BF, 32, 1), (HF, 64, 1), (BF, 128, 1), (HF, 32, 20), (BF, 64, 25)])
def test_split_keys_with_lengths(dt, D, T):
    """New tokens over caches of different lengths with several key splits a request (39, 32 and fewer: both forms of their
    join), splits without a key, sequences without one, and NaN behind the ends."""
    B, S, H, Hkv = 8, 5000, 4, 2
    q, k, v, lam, do = da_inputs(gen(300 + D), B, T, S, H, Hkv, D, dt)
    kv = torch.tensor([0, 1, 31, 33, 5000, 9999, 2600, 128], device="cuda", dtype=torch.int32)
    for b in range(B):
        k[b, min(S, int(kv[b])):] = math.nan
        v[b, min(S, int(kv[b])):] = math.nan
    out, (dq, dk, dv, _) = da_case(q, k, v, lam, do, causal=T == 1, kv_lens=kv)
    assert not out[0].any() and not dq[0].any() and not dk[2, 31:].any() and not dv[7, 128:].any()


@pytest.mark.parametrize("dt,D,causal,full", [(BF, 64, True, 600), (HF, 32, True, 600), (BF, 128, True, 600), (HF, 64, False, 600),
                                              (BF, 32, True, 640)])
def test_split_rows_with_lengths(dt, D, causal, full):
    """A padded training batch whose rows are split for dK and dV: splits that begin behind a short sequence's end, a sequence
    of no position, of a few, of fewer positions than keys; NaN behind the ends."""
    B, H, Hkv = 5, 4, 1
    T = S = full
    q, k, v, lam, do = da_inputs(gen(400 + D), B, T, S, H, Hkv, D, dt)
    lens = torch.tensor([0, full, 5, 333, 40], device="cuda", dtype=torch.int32)
    ql = torch.tensor([0, full, 5, 333, 7], device="cuda", dtype=torch.int32)
    for b in range(B):
        k[b, int(lens[b]):] = math.nan
        v[b, int(lens[b]):] = math.nan
        q[b, int(ql[b]):] = math.nan
    out, (dq, dk, dv, _) = da_case(q, k, v, lam, do, causal=causal, q_lens=ql, kv_lens=lens)
    assert not out[0].any() and not dk[0].any() and not dv[2, 5:].any() and not dq[4, 7:].any()


# ---------------------------------------------------------------------------------------------- Newton-Schulz
def structured(kind, m, n):
    g = gen(m + n)
    if kind == "signs":
        return torch.sign(randn(g, m, 1)) * torch.sign(randn(g, 1, n))
    if kind == "ones":
        return torch.ones(m, n, device="cuda")
    if kind == "thirds":
        return torch.full((m, n), 1 / 3, device="cuda")
    return randn(g, m, 3) @ randn(g, 3, n)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("kind", ["signs", "ones", "thirds", "rank 3"])
def test_newton_schulz_structured_matrices(kind, dt):
    """Matrices whose roundings do not average out, in every form (one workgroup, small and large tiles)."""
    import tossctr
    mats = [structured(kind, m, n).to(dt) for m, n in ((60, 90), (150, 333), (333, 150), (150, 500), (800, 1000))]
    for x, o in zip(mats, tossctr.newton_schulz(mats)):
        assert rel(o, ns_ref(x)) <= U[dt] + NS_TOL, tuple(x.shape)


@pytest.mark.parametrize("shape", [(96, 160), (150, 333), (800, 1000)])
def test_newton_schulz_16_bit_results_are_the_rounded_fp32_ones(shape):
    """Whatever the size, a 16-bit matrix is worked on as its fp32 copy is: the result is that one's rounding."""
    import tossctr
    for dt in (BF, HF):
        x = (randn(gen(5), *shape) * 1e-2).to(dt)
        got, want = tossctr.newton_schulz(x), tossctr.newton_schulz(x.float())
        assert torch.equal(got, want.to(dt))
