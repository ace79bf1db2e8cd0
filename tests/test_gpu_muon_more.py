"""FusedMuon beside the rest of a step: the EMA of the matrices during its warm-up, and data parallel over replicated and over
row-sharded tables (child processes whose two ranks share cuda:0 over gloo)."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
_cache = {}


def test_ema_of_the_matrices_follows_their_new_values():
    """shadow = d shadow + (1 - d) p with the decay of its warm-up and p as Muon left it: four fp32 roundings, each half a step of
    at most |shadow| + |p|."""
    from test_gpu_muon import trained
    from tossctr import FusedMuon
    from tossctr.optim import ema_decay_at
    model, opt, runs = trained(FusedMuon, 4)
    ema, ar, updates = opt.ema, model.arena, 0
    assert ema.warmup_steps > 0
    for i, (before, after, _, _, s0, s1) in enumerate(runs):
        due = ema.wants_update(i + 1)
        d = ema_decay_at(ema.base_decay, ema.warmup_steps, ema.warmup_type, updates)
        for k in opt.muon_params:
            p0, p, a, b = (ar._view(t, k).double() for t in (before, after, s0, s1))
            assert not torch.equal(p0, p)
            want = d * a + (1 - d) * p if due else a
            assert bool(((b - want).abs() <= 4 * 2.0 ** -24 * (a.abs() + p.abs())).all()), (i, k)
        updates += due
    assert updates == ema.num_updates > 1


def run(tmp_path_factory, worker, mode, same, steps=4, short=0):
    key = (worker, mode, same, steps, short)
    if key not in _cache:
        out = str(tmp_path_factory.mktemp("muon") / ("_".join(map(str, key)) + ".pt"))
        r = subprocess.run([sys.executable, os.path.join(HERE, f"dist_{worker}_worker.py"), "--mode", mode, "--same-batch", str(same),
                            "--steps", str(steps), "--short-last", str(short), "--out", out], capture_output=True, text=True, timeout=110)
        assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
        _cache[key] = torch.load(out, weights_only=True)
    return _cache[key]


def matrices(r):
    """The parameters that Muon took: AdamW's second moment of theirs never moved."""
    return [k for k in r["sd"] if r["sd"][k].dim() == 2 and not r["v"][k].any() and r["m"][k].any()]


@pytest.mark.parametrize("mode", ["replicated", "sharded"])
def test_momentum_is_of_the_clipped_mean_gradient(tmp_path_factory, mode):
    """After one step from zero AdamW's m is (1 - b1) times the clipped mean gradient of the ranks, Muon's is that gradient: equal
    but for two roundings, whatever the batches."""
    muon, adam = (run(tmp_path_factory, w, mode, 0, steps=1) for w in ("muon", "shard"))
    keys = matrices(muon)
    assert len(keys) > 5 and muon["gnorm"] == adam["gnorm"]
    for k in keys:
        a, b = muon["m"][k].double(), adam["m"][k].double() / (1 - 0.9)
        # m = fl(g (1 - 0.9f)): one rounding, and 1 - 0.9 in fp32 is within 2^-23 of 0.1
        assert bool(((a - b).abs() <= 2.0 ** -20 * a.abs() + 1e-37).all()), k


# Two ways to one gradient differ in the last bits of the clip's norm, so u by 2^-23 of itself; Newton-Schulz multiplies that by at
# most 3.4445^5 = 485 (6e-5 of O), the next gradients follow the parameters: held to 1e-4, as the other paths' outputs are
RTOL = 1e-4


def test_world2_of_one_batch_is_a_single_run(tmp_path_factory):
    from test_gpu_shard import _compare
    single = run(tmp_path_factory, "muon", "single", 1)
    for mode in ("replicated", "sharded"):
        _compare(run(tmp_path_factory, "muon", mode, 1), single, RTOL, what=f"{mode}: ")


@pytest.mark.parametrize("short", [0, 1])
def test_sharded_tables_match_replicated_ones(tmp_path_factory, short):
    from test_gpu_shard import _compare
    rep, sh = (run(tmp_path_factory, "muon", m, 0, short=short) for m in ("replicated", "sharded"))
    assert sh["local_rows"] == (sh["vocab"] + 1) // 2 and rep["local_rows"] == rep["vocab"]
    assert matrices(rep) == matrices(sh)
    _compare(sh, rep, RTOL, what="sharded: ")
