"""A ``train.optimizer`` that names no optimizer is taken for AdamW, and not in silence (no GPU)."""
import warnings

import pytest

from tossctr import optim


def build(monkeypatch, **train):
    made = []
    monkeypatch.setattr(optim, "FusedMuon", lambda *a, **k: made.append("muon"))
    monkeypatch.setattr(optim, "FusedAdamW", lambda *a, **k: made.append("adamw"))
    optim.build_optimizer(None, {"train": dict({"lr": 1e-3, "weight_decay": 0.1}, **train)})
    return made


@pytest.mark.parametrize("name", ["mu0n", "moun", "adam", "sgd", 3])
def test_other_names_warn(monkeypatch, name):
    with pytest.warns(UserWarning, match="neither 'adamw' nor 'muon'"):
        assert build(monkeypatch, optimizer=name) == ["adamw"]


@pytest.mark.parametrize("train,made", [({}, "adamw"), ({"optimizer": None}, "adamw"), ({"optimizer": "AdamW"}, "adamw"),
                                        ({"optimizer": "muon"}, "muon"), ({"optimizer": "MUON"}, "muon")])
def test_known_names_do_not(monkeypatch, train, made):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert build(monkeypatch, **train) == [made]


@pytest.mark.parametrize("config", ["dare_base", "dare_qnn_next", "v3_k148_s1", "hb1e8_d64"])
def test_muon_takes_no_bias_and_no_looked_up_row(config):
    """Of every config's parameters: matrices that multiply, none of those that are added or looked up (num_embed.bias has a row a
    feature, and is no matrix for that)."""
    from oracle.model import make_arch
    from tossctr import configs
    cfg = getattr(configs, config)()
    cards = configs.cat_cardinals(cfg)
    shapes = dict(make_arch(cfg, 1000, configs.N_NUM_NEXT, configs.N_NUM_NEXT, cards, list(cards)).param_shapes())
    kind = {k: "table" if k.startswith("cat_embs.") or ".emb_" in k else "dense" for k in shapes}
    keys = optim.muon_keys(list(shapes), shapes, kind, len(shapes), {k: i for i, k in enumerate(shapes)})
    assert len(shapes["num_embed.bias"]) == 2 and "num_embed.out_proj.weight" in keys
    assert not [k for k in keys if "bias" in k or k in ("num_embed.weight", "mask_embed.weight") or kind[k] != "dense"]
