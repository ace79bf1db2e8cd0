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
