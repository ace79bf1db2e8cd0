"""Measured operators of a differential-attention encoder block: layer norm (forward, backward and the weight's
gradient), differential attention (training, prefill, single tokens over a cache) and the Newton-Schulz
orthogonalisation that a Muon update takes of its weight matrices.

``own = False`` computes them in plain torch operations; ``own = True`` calls the framework's entry points."""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
LN_EPS = 1e-5


@functools.lru_cache(maxsize=None)
def _tossctr():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "toss-next-ctr-prediction_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import tossctr
    return tossctr


# ---------------------------------------------------------------------------------------------- cases
def _ln(name, rows, width, dtype, train):
    return {"name": name, "op": "ln", "rows": rows, "width": width, "dtype": dtype, "train": train}


def _ns(name, shapes, dtype):
    return {"name": name, "op": "ns", "shapes": shapes, "dtype": dtype}


def _da(name, B, T, S, H, Hkv, d, dtype, causal, ragged, train):
    return {"name": name, "op": "da", "B": B, "T": T, "S": S, "H": H, "Hkv": Hkv, "d": d, "dtype": dtype,
            "causal": causal, "ragged": ragged, "train": train}


def listed():
    return [
        # a fine-tuning micro-batch of a few tokens: launches and host time count
        _ln("ln small", 64, 256, "bf16", True),
        # serving: the pre-norm of a ragged batch of tokens, a width that no vector divides
        _ln("ln odd serving", 4099, 1001, "fp16", False),
        # the encoder's norms at batch 4096 and 60 selected events of width 32
        _ln("ln encoder rows", 245760, 32, "bf16", True),
        # the pre-norm of a wide model over a large token batch
        _ln("ln wide", 32768, 4096, "bf16", True),
        # the matrices of three encoder layers at width 32 (in-projection, out-projection, FFN up and down)
        _ns("ns encoder", ",".join(["96x32", "32x32", "384x32", "32x384"] * 3), "fp32"),
        # the first matrix of the interaction MLP, fp32 master gradient
        _ns("ns mlp", "512x7552", "fp32"),
        # a feed-forward matrix of a wide model, bf16 gradient
        _ns("ns ffn", "2048x8192", "bf16"),
        # an encoder step over 60 selected events, every event sees every other
        _da("da encoder", 32, 60, 60, 4, 4, 32, "bf16", False, False, True),
        # a causal training step on a padded batch of long histories with shared key heads
        _da("da train", 2, 4096, 4096, 16, 4, 64, "bf16", True, True, True),
        # a prefill chunk behind a cache that is there already, odd lengths
        _da("da prefill", 1, 1531, 5627, 16, 8, 128, "fp16", True, False, False),
        # one new token for each of many requests, caches of different lengths
        _da("da decode", 48, 1, 4096, 16, 4, 64, "bf16", False, True, False),
        # one new token over one very long cache
        _da("da decode long", 1, 1, 131072, 8, 2, 128, "bf16", False, False, False),
    ]


def _logu(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _odd(rng, lo, hi):
    """A size spread over its logarithm: any whole number two times in three, else a multiple of 16."""
    n = _logu(rng, lo, hi)
    return n if n < 32 or rng.random() < 2 / 3 else n // 16 * 16


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("ln", "ns", "da")}
    pairs = max(c["B"] * c["H"] * c["T"] * c["S"] for c in listed() if c["op"] == "da")
    while True:
        op = rng.choice(["ln", "ns", "da", "da"])
        if op == "ln":
            c = _ln("", _odd(rng, 1, 262144), _odd(rng, 16, 8192), rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.7)
        elif op == "ns":
            n = rng.choice([1, 1, 2, 5])
            c = _ns("", ",".join("%dx%d" % (_odd(rng, 16, 4096), _odd(rng, 16, 8192)) for _ in range(n)),
                    rng.choice(["fp32", "bf16", "fp16"]))
        else:
            kind = rng.choice(["train", "train", "prefill", "decode", "decode"])
            Hkv, G, d = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 128])
            dt = rng.choice(["bf16", "fp16"])
            if kind == "train":
                T = _odd(rng, 16, 4096)
                c = _da("", _logu(rng, 1, 64), T, T, Hkv * G, Hkv, d, dt, rng.random() < 0.6, rng.random() < 0.5, True)
            elif kind == "prefill":
                T = _odd(rng, 2, 4096)
                c = _da("", _logu(rng, 1, 8), T, T + rng.choice([0, 1]) * _odd(rng, 1, 8192), Hkv * G, Hkv, d, dt, True,
                        False, False)
            else:
                c = _da("", _logu(rng, 1, 64), 1, _odd(rng, 16, 131072), Hkv * G, Hkv, d, dt, False, rng.random() < 0.7,
                        False)
            if c["B"] * c["H"] * c["T"] * c["S"] > pairs or c["B"] * c["S"] * c["Hkv"] * c["d"] > 1 << 28:
                continue
        c.pop("name")
        if _cost(c) <= most[op]:
            return c


# ---------------------------------------------------------------------------------------------- inputs
def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device=dev, generator=g, dtype=torch.float32)

    if case["op"] == "ln":
        M, N = case["rows"], case["width"]
        # activations of a residual stream: a spread per row and a mean that is not zero; master weights in fp32
        x = (randn(M, N) * (0.5 + randn(M, 1).abs()) + 0.3 * randn(M, 1)).to(dt)
        return {"op": "ln", "train": case["train"], "x": x, "dy": randn(M, N).to(dt), "w": 1 + 0.1 * randn(N),
                "b": 0.1 * randn(N)}
    if case["op"] == "ns":
        # momentum of gradients: noise and a few strong directions
        mats = [(randn(m, n) + 4 * randn(m, 2) @ randn(2, n) / 2 ** 0.5).mul_(1e-3).to(dt) for m, n in _shapes(case)]
        return {"op": "ns", "mats": mats}
    B, T, S, H, Hkv, d = (case[k] for k in ("B", "T", "S", "H", "Hkv", "d"))
    st = {"op": "da", "train": case["train"], "causal": case["causal"],
          "q": randn(B, T, H, 2, d).to(dt), "k": randn(B, S, Hkv, 2, d).to(dt), "v": randn(B, S, Hkv, 2 * d).to(dt),
          "lam": 0.2 + 0.6 * torch.rand(H, device=dev, generator=g), "lens": None}
    if case["train"]:
        st["do"] = randn(B, T, H, 2 * d).to(dt)
    if case["ragged"]:
        # one sequence of the whole length, the others between an eighth of it and the whole
        lens = torch.randint(max(1, S // 8), S + 1, (B,), device=dev, generator=g, dtype=torch.int32)
        lens[0] = S
        st["lens"] = lens
    return st


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_ln(st):
    x, w, b = st["x"].float(), st["w"], st["b"]
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + LN_EPS)
    xhat = xc * rstd
    y = (xhat * w + b).to(st["x"].dtype)
    if not st["train"]:
        return y
    dy = st["dy"].float()
    gw = dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    dw = (dy * xhat).sum(0, dtype=torch.float64).float()
    db = dy.sum(0, dtype=torch.float64).float()
    return y, dx.to(st["x"].dtype), dw, db


def _plain_ns_one(mat):
    a, b, c = NS_COEFFS
    x = mat.float()
    wide = x if x.shape[0] <= x.shape[1] else x.t()
    x = wide / (wide.double().square().sum().sqrt() + NS_EPS).float()

    def once(x, _):
        g = x @ x.t()
        return a * x + (b * g + c * (g @ g)) @ x

    x = functools.reduce(once, range(NS_STEPS), x)
    return (x if mat.shape[0] <= mat.shape[1] else x.t()).to(mat.dtype)


def _seen(st, B, T, S, dev):
    """(B, 1, 1, 1, T, S): which keys a row sees -- those before its sequence's end and, causally, not after it when
    the sequence's last row and last key stand level; rows behind the end see none."""
    j, i = torch.arange(S, device=dev), torch.arange(T, device=dev)
    kl = st["lens"].long() if st["lens"] is not None else torch.full((B,), S, device=dev)
    ql = kl if (st["lens"] is not None and T > 1) else torch.full((B,), T, device=dev)
    seen = (j[None, None, :] < kl[:, None, None]) & (i[None, :, None] < ql[:, None, None])
    if st["causal"]:
        seen = seen & (j[None, None, :] <= (i[None, :] + (kl - ql)[:, None])[:, :, None])
    return seen[:, None, None, None]


def _plain_da(st):
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    B, T, H, _, d = q.shape
    S, Hkv = k.shape[1], k.shape[2]
    G, dt, scale = H // Hkv, st["q"].dtype, 1.0 / math.sqrt(d)
    q = q.view(B, T, Hkv, G, 2, d).permute(0, 2, 3, 4, 1, 5)             # B Hkv G 2 T d
    k = k.permute(0, 2, 3, 1, 4).unsqueeze(2)                            # B Hkv 1 2 S d
    v = v.permute(0, 2, 1, 3)[:, :, None, None]                          # B Hkv 1 1 S dv
    lam = st["lam"].view(Hkv, G)[None, :, :, None, None]
    seen = _seen(st, B, T, S, q.device)
    s = torch.where(seen, (q @ k.transpose(-1, -2)) * scale, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    del s
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ v                                                            # B Hkv G 2 T dv
    o1, o2 = o[:, :, :, 0], o[:, :, :, 1]
    out = (o1 - lam * o2).permute(0, 3, 1, 2, 4).reshape(B, T, H, -1).to(dt)
    if not st["train"]:
        return out
    do = st["do"].float().view(B, T, Hkv, G, -1).permute(0, 2, 3, 1, 4)  # B Hkv G T dv
    sign = torch.stack([torch.ones_like(lam), -lam], 3)                  # B' Hkv G 2 1 1
    delta = torch.stack([(do * o1).sum(-1), (do * o2).sum(-1)], 3).unsqueeze(-1)
    dp = (do @ v[:, :, :, 0].transpose(-1, -2)).unsqueeze(3)             # B Hkv G 1 T S
    dv = ((p[:, :, :, 0] - lam * p[:, :, :, 1]).transpose(-1, -2) @ do).sum(2)
    ds = p * (dp - delta) * (sign * scale)
    del p, dp
    dq = (ds @ k).permute(0, 4, 1, 2, 3, 5).reshape(B, T, H, 2, d)
    dk = (ds.transpose(-1, -2) @ q).sum(2).permute(0, 3, 1, 2, 4)
    dlam = -delta[:, :, :, 1, :, 0].sum((0, 3), dtype=torch.float64).float().reshape(H)
    return out, dq.to(dt), dk.to(dt), dv.permute(0, 2, 1, 3).to(dt), dlam


def run(st):
    if own:
        t = _tossctr()
        if st["op"] == "ln":
            y, mean, rstd = t.layer_norm_fwd(st["x"], st["w"], st["b"], LN_EPS)
            if not st["train"]:
                return y
            return (y, *t.layer_norm_bwd(st["dy"], st["x"], mean, rstd, st["w"]))
        if st["op"] == "ns":
            return t.newton_schulz(st["mats"], steps=NS_STEPS, coeffs=NS_COEFFS, eps=NS_EPS)
        q, k, v, lam, lens = st["q"], st["k"], st["v"], st["lam"], st["lens"]
        mask = {"causal": st["causal"], "kv_lens": lens, "q_lens": lens if q.shape[1] > 1 else None}
        if not st["train"]:
            return t.diff_attention_fwd(q, k, v, lam, save=False, **mask)[0]
        out, saved = t.diff_attention_fwd(q, k, v, lam, **mask)
        return (out, *t.diff_attention_bwd(st["do"], q, k, v, lam, out, saved, **mask))
    if st["op"] == "ln":
        return _plain_ln(st)
    if st["op"] == "ns":
        return [_plain_ns_one(m) for m in st["mats"]]
    return _plain_da(st)


# ---------------------------------------------------------------------------------------------- work, exact values
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "ln":
        M, N = case["rows"], case["width"]
        # x and y; with the backward pass dy and dx, the weight, the bias and their gradients
        return {"bytes": M * N * e * (4 if case["train"] else 2) + 4 * N * (4 if case["train"] else 2),
                "flops": M * N * (22 if case["train"] else 8)}
    if case["op"] == "ns":
        dims = [(min(s), max(s)) for s in _shapes(case)]
        # X X^T and its square are symmetric: half of their products; the last one is whole
        return {"bytes": sum(2 * m * n * e for m, n in dims),
                "flops": sum(NS_STEPS * (m * m * n + m ** 3 + 2 * m * m * n) for m, n in dims)}
    B, T, S, H, Hkv, d = (case[k] for k in ("B", "T", "S", "H", "Hkv", "d"))
    share = 1.0
    if case["ragged"]:        # lengths between S / 8 and S
        share = 0.36 if T > 1 else 0.57
    seen = B * H * share * ((T * S - T * (T - 1) / 2) if case["causal"] else T * S)
    cache = share ** 0.5 if T > 1 else share
    qo, kv = B * T * H * 2 * d, cache * B * S * Hkv * 4 * d
    # two maps of width d, two products with the values of width 2d; backward: dP, dV, and dQ, dK of either map,
    # after the maps again
    flops = seen * (2 * 2 * d + 2 * 2 * 2 * d) + (seen * (2 * 2 * d + 2 * 2 * d * 2 + 4 * 2 * d) if case["train"] else 0)
    return {"bytes": e * (2 * qo + kv) * (2 if case["train"] else 1), "flops": flops}


def exact(case, seed):
    """From the definitions in 64 bits: gradients by differentiating the definition, the orthogonalisation as a
    polynomial of the Gram matrix alone."""
    st = prepare(case, seed)
    if st["op"] == "ln":
        x, w, b = (st[n].double().requires_grad_() for n in ("x", "w", "b"))
        y = torch.nn.functional.layer_norm(x, (x.shape[-1],), w, b, LN_EPS)
        if not st["train"]:
            return y.detach()
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), st["dy"].double()))
    if st["op"] == "ns":
        def orthogonal(g):
            a, b, c = NS_COEFFS
            wide = g if g.shape[0] <= g.shape[1] else g.t()
            x = wide / (torch.linalg.vector_norm(wide) + NS_EPS)
            eye = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
            gram, q = x @ x.t(), eye
            for _ in range(NS_STEPS):       # X_k = Q_k X, Gram_k = Q_k Gram Q_k
                p = a * eye + b * gram + c * (gram @ gram)
                q, gram = p @ q, p @ gram @ p
            x = q @ x
            return x if g.shape[0] <= g.shape[1] else x.t()

        return [orthogonal(m.double()) for m in st["mats"]]
    with torch.enable_grad():
        q, k, v, lam = (st[n].double().requires_grad_(st["train"]) for n in ("q", "k", "v", "lam"))
        B, T, H, _, d = q.shape
        S, Hkv = k.shape[1], k.shape[2]
        seen = _seen(st, B, T, S, q.device)[:, :, 0, 0]
        vv = v.repeat_interleave(H // Hkv, 2).transpose(1, 2)

        def one(c):
            kk = k[:, :, :, c].repeat_interleave(H // Hkv, 2).permute(0, 2, 3, 1)
            s = (q[:, :, :, c].transpose(1, 2) @ kk / math.sqrt(d)).masked_fill(~seen, -1e300)
            return s.softmax(-1).masked_fill(~seen, 0.0) @ vv

        out = (one(0) - lam[:, None, None] * one(1)).transpose(1, 2)
        if not st["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (q, k, v, lam), st["do"].double()))
