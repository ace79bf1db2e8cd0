"""FusedMuon: the Muon rule on the dense matrices against its definition in 64 bits, everything else FusedAdamW's bits, and
the K-fold loop with ``train.optimizer: muon``."""
import os
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_ops import NS_TOL, ns_ref  # noqa: E402


def trained(cls, steps, **kw):
    """[(params before, params after, dense grads, clip multiplier, EMA shadow before and after)] of `steps` fused steps."""
    from golden_util import Fixture
    from tossctr import CTRModel, build_ema
    fx = Fixture("tiny_concat")
    m = fx.meta
    model = CTRModel(m["cfg"], m["vocab"], m["Fn"], m["Fm"], fx.cat_cards, fx.cat_cols, device="cuda:0")
    model.load_state_dict({k: torch.from_numpy(v) for k, v in fx.params0().items()})
    ema = build_ema(model, m["cfg"])
    tr = m["train"]
    opt = cls(model, lr=1e-2, weight_decay=0.1, max_grad_norm=tr["clip"], ema=ema, **kw)
    out = []
    for i in range(steps):
        b = fx.batch(0)
        inputs = model.stage({k: torch.from_numpy(b[k]) for k in ("X_num", "X_mask", "X_cat", "seq")})
        y = torch.from_numpy(b["y"]).float().cuda()
        model.sync()
        before, sh0 = model.arena.buf.clone(), ema.shadow.clone() if ema else None
        model.train_step(inputs, y, opt, global_step=i + 1, seed=m["seeds"][0])
        model.sync()
        torch.cuda.synchronize()
        out.append((before, model.arena.buf.clone(), model.arena.grad.clone(), float(opt.norm_out[1]), sh0,
                    ema.shadow.clone() if ema else None))
    return model, opt, out


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps(nesterov):
    from tossctr import FusedAdamW, FusedMuon
    lr, wd, mu = 1e-2, 0.1, 0.95
    model, opt, runs = trained(FusedMuon, 3, nesterov=nesterov, momentum=mu)
    ar = model.arena
    assert opt.muon_params and all(len(ar.shapes[k]) == 2 for k in opt.muon_params)
    assert any("in_proj_weight" in k for k in opt.muon_params) and any("ffn.0" in k for k in opt.muon_params)
    for k in opt.muon_params:
        view = lambda t: ar._view(t, k).double()  # noqa: E731
        buf = 0.0
        for before, after, grad, coef, *_ in runs:
            g = view(grad) * coef
            buf = mu * buf + g
            o = ns_ref(g + mu * buf if nesterov else buf)
            want = (1 - lr * wd) * view(before) - lr * 0.2 * max(ar.shapes[k]) ** 0.5 * o
            # u's three fp32 roundings go through the iteration as its own do; p's two are half a step of it each
            tol = lr * 0.2 * max(ar.shapes[k]) ** 0.5 * 2 * NS_TOL * o.norm() + 2 * 2.0 ** -24 * view(before).norm()
            assert float((view(after) - want).norm()) <= float(tol), k
    # the rest of the first step is FusedAdamW's, bit for bit (later ones see other matrices)
    base, _, ref = trained(FusedAdamW, 1)
    taken = torch.zeros_like(runs[0][1], dtype=torch.bool)
    for k in opt.muon_params:
        ar._view(taken, k).fill_(True)
    assert torch.equal(runs[0][0], ref[0][0]) and torch.equal(runs[0][2], ref[0][2])
    assert torch.equal(runs[0][1][~taken], ref[0][1][~taken]) and not torch.equal(runs[0][1][taken], ref[0][1][taken])
    if runs[0][5] is not None:           # the EMA of the matrices moves with their new values
        d = opt.ema.base_decay if opt.ema.warmup_steps <= 0 else None
        if d is not None:
            before, after, _, _, s0, s1 = runs[0]
            want = d * s0.double() + (1 - d) * after.double()
            assert float((s1.double() - want)[taken].abs().max()) <= 2.0 ** -22 * float(after.abs().max() + s0.abs().max())


def test_muon_refusals():
    from golden_util import Fixture
    from tossctr import CTRModel, FusedMuon
    fx = Fixture("tiny_concat")
    m = fx.meta
    model = CTRModel(m["cfg"], m["vocab"], m["Fn"], m["Fm"], fx.cat_cards, fx.cat_cols, device="cuda:0")
    with pytest.raises(ValueError, match="momentum"):
        FusedMuon(model, lr=1e-3, momentum=1.0)
    with pytest.raises(ValueError, match="ns_steps"):
        FusedMuon(model, lr=1e-3, ns_steps=0)


def test_kfold_loop_with_muon(tmp_path):
    from test_gpu_train import tiny_run_cfg
    from tossctr.data import synth_rows, write_shard_cache
    from tossctr.train import main
    arr = synth_rows(2000, 6, 6, [203, 203, 203, 203], 24, 3000, seed=5, pos_rate=0.2)
    man = write_shard_cache(str(tmp_path / "cache"), arr, shard_rows=1100, num_cols=[f"n{i}" for i in range(6)],
                            cat_cols=["c0", "c1", "c2", "c3"], group_key="c0")
    cfg = tiny_run_cfg(str(tmp_path), man)
    cfg["train"]["optimizer"] = "muon"
    res = main(cfg)
    assert list(res) == [0] and np.isfinite(res[0])
