"""Refusals of layer norm, differential attention and Newton-Schulz: in Python, and at the C entries (which check before
any launch, so they need no GPU)."""
import ctypes as C

import pytest
import torch

import tossctr
from tossctr import _lib

BF = torch.bfloat16


def z(*s, dt=BF):
    return torch.zeros(*s, dtype=dt)


@pytest.mark.parametrize("call,error,match", [
    (lambda: tossctr.layer_norm_fwd(z(3, 0), z(0)), ValueError, "at least one element"),
    (lambda: tossctr.layer_norm_fwd(z(3, 8, dt=torch.float64), z(8)), TypeError, "float64"),
    (lambda: tossctr.layer_norm_fwd(z(3, 8), z(7)), ValueError, "weight of shape"),
    (lambda: tossctr.layer_norm_fwd(z(3, 8), z(8, dt=torch.float16)), TypeError, "weight in float32"),
    (lambda: tossctr.layer_norm_fwd(z(3, 8), z(8), z(8, dt=torch.float32)), TypeError, "bias in float32"),
    (lambda: tossctr.layer_norm_fwd(z(3, 8), z(8)), ValueError, "device tensors"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 2, 32), z(1, 4, 2, 2, 32), z(1, 4, 2, 64), z(2)), ValueError, "q of shape"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 2, 2, 32), z(2, 4, 2, 2, 32), z(1, 4, 2, 64), z(2)), ValueError, "k of shape"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 2, 2, 32), z(1, 4, 2, 2, 32), z(1, 4, 2, 32), z(2)), ValueError, "v of shape"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 2, 2, 48), z(1, 4, 2, 2, 48), z(1, 4, 2, 96), z(2)), NotImplementedError,
     "width 32, 64 or 128"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 3, 2, 32), z(1, 4, 2, 2, 32), z(1, 4, 2, 64), z(3)), ValueError,
     "3 query heads over 2"),
    (lambda: tossctr.diff_attention_fwd(*(z(*s, dt=torch.float32) for s in ((1, 4, 2, 2, 32), (1, 4, 2, 2, 32), (1, 4, 2, 64))),
                                        z(2)), TypeError, "bfloat16 or float16"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 2, 2, 32), z(1, 4, 2, 2, 32, dt=torch.float16), z(1, 4, 2, 64), z(2)),
     TypeError, "one type"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 2, 2, 32), z(1, 4, 2, 2, 32), z(1, 4, 2, 64), z(2)), ValueError, "lam of 2 float32"),
    (lambda: tossctr.diff_attention_fwd(z(1, 4, 2, 2, 32), z(1, 4, 2, 2, 32), z(1, 4, 2, 64), z(2, dt=torch.float32)),
     ValueError, "device tensors"),
    (lambda: tossctr.newton_schulz(z(5)), ValueError, "matrices"),
    (lambda: tossctr.newton_schulz([z(2, 3, 4)]), ValueError, "matrices"),
    (lambda: tossctr.newton_schulz([z(3, 4), z(3, 4, dt=torch.float32)]), TypeError, "for all"),
    (lambda: tossctr.newton_schulz(z(3, 4)), ValueError, "device tensors"),
])
def test_python_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


P = 1 << 20        # an aligned address that nothing dereferences


def refuse(match, name, *args):
    with pytest.raises(_lib.CtrError, match=match):
        _lib.call(name, *args)


def test_ln_entry_refusals():
    fwd = lambda m=4, n=8, ldx=8, ldy=8, xt=1, wt=0, x=P, mean=P: (  # noqa: E731
        x, ldx, m, n, P, P, 1e-5, P, ldy, mean, P, xt, wt, None)
    refuse("sizes", "ctr_ln_fwd", *fwd(m=-1))
    refuse("sizes", "ctr_ln_fwd", *fwd(n=0))
    refuse("row strides", "ctr_ln_fwd", *fwd(ldy=7))
    refuse("null operand", "ctr_ln_fwd", *fwd(x=None))
    refuse("types", "ctr_ln_fwd", *fwd(xt=1, wt=2))
    refuse("types", "ctr_ln_fwd", *fwd(xt=3))
    assert _lib.call("ctr_ln_fwd", *fwd(m=0)) == 0
    need = _lib.query("ctr_ln_bwd_ws_size", 1000, 64)
    assert need > 0 and _lib.query("ctr_ln_bwd_ws_size", 0, 64) == 0
    bwd = lambda ws=need, dw=P, lddx=64: (  # noqa: E731
        P, 64, P, 64, P, P, P, 1000, 64, P, lddx, dw, P, P, ws, 1, 0, None)
    refuse("workspace", "ctr_ln_bwd", *bwd(ws=need - 1))
    refuse("null operand", "ctr_ln_bwd", *bwd(dw=None))
    refuse("row strides", "ctr_ln_bwd", *bwd(lddx=63))


def attn(**kw):
    a = _lib.DiffAttn()
    for f in ("q", "k", "v", "lam", "o", "o2", "ol", "stat"):
        setattr(a, f, P)
    B, T, S, H, Hkv, D = 2, 64, 64, 4, 2, 64
    a.q_sb, a.q_st, a.q_sh, a.q_sc = T * H * 2 * D, H * 2 * D, 2 * D, D
    a.k_sb, a.k_ss, a.k_sh, a.k_sc = S * Hkv * 2 * D, Hkv * 2 * D, 2 * D, D
    a.v_sb, a.v_ss, a.v_sh = S * Hkv * 2 * D, Hkv * 2 * D, 2 * D
    a.scale, a.B, a.T, a.S, a.H, a.Hkv, a.D, a.causal, a.type = 0.125, B, T, S, H, Hkv, D, 0, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,match", [
    ({"type": 0}, "type"), ({"D": 48}, "map width"), ({"H": 3}, "sizes"), ({"Hkv": 0}, "sizes"), ({"T": -1}, "sizes"),
    ({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"lam": None}, "null lam"), ({"q": P + 8}, "q: 16-byte"),
    ({"q_st": 4}, "q: 16-byte"), ({"k_sc": 63}, "k: 16-byte"), ({"v": None}, "v: 16-byte"), ({"o": None}, "output"),
    ({"T": 1 << 29}, "sizes"), ({"B": 1 << 20, "T": 1 << 12}, "sizes")])
def test_diffattn_entry_refusals(kw, match):
    refuse(match, "ctr_diffattn_fwd", C.byref(attn(**kw)), P, 1 << 40, None)
    refuse(match, "ctr_diffattn_bwd", C.byref(attn(**kw)), P, 64, 64, 64, P, P, P, P, P, 1 << 40, None)


def test_diffattn_entry_workspaces_and_gradients():
    a = attn(T=1, S=1 << 16)
    need = _lib.query("ctr_diffattn_fwd_ws_size", C.byref(a))
    assert need > 0
    refuse("workspace", "ctr_diffattn_fwd", C.byref(a), P, need - 1, None)
    a = attn()
    need = _lib.query("ctr_diffattn_bwd_ws_size", C.byref(a))
    good = lambda **kw: [C.byref(a)] + [kw.get(k, v) for k, v in (("g", P), ("sb", 64), ("st", 64), ("sh", 64), ("dq", P),  # noqa: E731
                                        ("dk", P), ("dv", P), ("dlam", P), ("ws", P), ("n", need), ("s", None))]
    refuse("workspace", "ctr_diffattn_bwd", *good(n=need - 1))
    refuse("null dlam", "ctr_diffattn_bwd", *good(dlam=None))
    refuse("dout", "ctr_diffattn_bwd", *good(st=4))
    refuse("null operand", "ctr_diffattn_bwd", *good(dk=None))
    refuse("16-byte", "ctr_diffattn_bwd", *good(dq=P + 2))
    b = attn(o2=None, ol=None)
    refuse("null operand", "ctr_diffattn_bwd", C.byref(b), *good()[1:])
    assert _lib.call("ctr_diffattn_fwd", C.byref(attn(B=0)), None, 0, None) == 0


def test_diffattn_head_strides_stay_within_32_bit_offsets():
    """A tile addresses a group's heads by 32-bit byte offsets: 100 heads of 2^23 elements are beyond them, 2 are not."""
    for heads, st in ((100, 1 << 23), (2, 1 << 30)):
        refuse("q: 16-byte", "ctr_diffattn_fwd", C.byref(attn(H=heads, Hkv=1, q_sh=st)), P, 0, None)
        a = attn(H=heads, Hkv=1)
        refuse("dout", "ctr_diffattn_bwd", C.byref(a), P, 64, 64, st, P, P, P, P, P, 1 << 40, None)
    refuse("workspace", "ctr_diffattn_bwd", C.byref(attn(H=2, Hkv=1, q_sh=1 << 23)), P, 64, 64, 1 << 23, P, P, P, P, P, 0, None)
    from tossctr.ops import _aligned
    t = torch.empty_strided((1, 2, 100, 2, 32), (8, 64, 1 << 23, 32, 1), dtype=BF, device="meta")
    r, st = _aligned(t)
    assert r is not t and st[2] == 64


def test_newton_schulz_entry_refusals():
    def mats(rows=300, cols=400, ld=400, src=P, dst=P):
        arr = (_lib.NsMat * 1)()
        arr[0].src, arr[0].dst, arr[0].ld_src, arr[0].ld_dst, arr[0].rows, arr[0].cols = src, dst, ld, ld, rows, cols
        return arr

    ok = (5, 3.4445, -4.7750, 2.0315, 1e-7, 0)
    need = _lib.query("ctr_newton_schulz_ws_size", mats(), 1)
    assert need > 0 and _lib.query("ctr_newton_schulz_ws_size", mats(32, 32, 32), 1) == 0
    refuse("workspace", "ctr_newton_schulz", mats(), 1, *ok, P, need - 1, None)
    refuse("row strides", "ctr_newton_schulz", mats(ld=399), 1, *ok, P, need, None)
    refuse("null matrix", "ctr_newton_schulz", mats(dst=None), 1, *ok, P, need, None)
    refuse("sides", "ctr_newton_schulz", mats(rows=1 << 20), 1, *ok, P, 1 << 50, None)
    refuse("type", "ctr_newton_schulz", mats(), 1, *ok[:5], 3, P, need, None)
    refuse("steps", "ctr_newton_schulz", mats(), 1, 0, *ok[1:], P, need, None)
    refuse("eps", "ctr_newton_schulz", mats(), 1, *ok[:4], -1.0, 0, P, need, None)
    for c in ((40.0, 0.0, 0.0), (3.0, 3.0, 3.0), (float("nan"), 0.0, 0.0), (2.0, 0.0, 0.0)):
        refuse("coefficients", "ctr_newton_schulz", mats(), 1, 5, *c, 1e-7, 0, P, need, None)
    assert _lib.call("ctr_newton_schulz", None, 0, *ok, None, 0, None) == 0


@pytest.mark.parametrize("make,copied", [
    (lambda: z(2, 5, 3, 2, 32), False),
    (lambda: z(2, 5, 6, 2, 32)[:, 1:4, ::2], False),
    (lambda: z(1, 5, 3, 2, 32).expand(4, 5, 3, 2, 32), False),          # one batch for all
    (lambda: z(2, 5, 3, 2, 64)[..., ::2], True),
    (lambda: z(2, 5, 3, 2, 33)[..., :32], True),                         # rows off the 16 bytes
    (lambda: z(1).expand(2, 5, 3, 2, 32), True),                         # the gradient of a sum: one element for all
    (lambda: z(2, 5, 3, 2, 1).expand(2, 5, 3, 2, 32), True)])
def test_attention_rows_read_in_place_or_copied(make, copied):
    from tossctr.ops import _aligned
    t = make()
    r, st = _aligned(t)
    assert (r is not t) == copied and r.shape == t.shape
    assert r.stride(-1) == 1 and all(s % 8 == 0 for s in st) and list(st) == [s if n > 1 else 0 for s, n in zip(r.stride(), r.shape)][:-1]
