"""Which parameters FusedMuon takes, and how ``train.optimizer`` names it (no GPU)."""
import ctypes as C

import pytest

from tossctr import _lib, optim


def test_muon_keys():
    shapes = {"num_embed.weight": (6, 8), "num_embed.out_proj.weight": (16, 8), "mask_embed.weight": (6, 8),
              "cat_embs.c0.weight": (200, 8), "cat_proj.c0.weight": (16, 8), "dare.layers.0.mha.in_proj_weight": (48, 16),
              "dare.layers.0.mha.in_proj_bias": (48,), "dare.layers.0.pbias.rel.weight": (25, 4), "qnn.U": (2, 16, 4),
              "qnn.mlp.6.weight": (1, 16), "ctx_mlp.0.weight": (16, 48)}
    kind = {k: "table" if k.startswith("cat_embs.") else "dense" for k in shapes}
    offs = {k: 64 * i for i, k in enumerate(shapes)}
    keys = optim.muon_keys(list(shapes), shapes, kind, 64 * (len(shapes) - 1), offs)      # the last has no gradient
    assert keys == ["num_embed.out_proj.weight", "cat_proj.c0.weight", "dare.layers.0.mha.in_proj_weight"]


def test_build_optimizer_names(monkeypatch):
    made = []
    monkeypatch.setattr(optim, "FusedMuon", lambda *a, **k: made.append(("muon", k)))
    monkeypatch.setattr(optim, "FusedAdamW", lambda *a, **k: made.append(("adamw", k)))
    tr = {"lr": 1e-3, "weight_decay": 0.1}
    optim.build_optimizer(None, {"train": dict(tr, optimizer="muon")})
    optim.build_optimizer(None, {"train": dict(tr, optimizer="adamw", grad_clip_norm=0.5)})
    optim.build_optimizer(None, {"train": tr})
    assert [m[0] for m in made] == ["muon", "adamw", "adamw"] and made[1][1]["max_grad_norm"] == 0.5


def test_muon_entry_refusals():
    arr = (_lib.MuonMat * 1)()
    arr[0].n = 4
    with pytest.raises(_lib.CtrError, match="null matrix"):
        _lib.call("ctr_muon_update", arr, 1, 1, None, 0.9, 1, 0.1, 0.0, None)
    with pytest.raises(_lib.CtrError, match="null coefficient"):
        _lib.call("ctr_muon_update", arr, 1, 0, None, 0.9, 1, 0.1, 0.0, None)
    with pytest.raises(_lib.CtrError, match="matrix list"):
        _lib.call("ctr_muon_update", C.POINTER(_lib.MuonMat)(), 1, 1, None, 0.9, 1, 0.1, 0.0, None)
    assert arr[0].n == 4
