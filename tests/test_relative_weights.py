"""Weights that encoders with relative positions start from and are trained to: what is loaded and what is refused."""
import dataclasses

import pytest
import torch

from renee_b200.cli import build_parser, start
from renee_b200.models.encoder import DistilEncoder, EncoderConfig, load_initial_weights
from renee_b200.models.flat_encoder import FlatEncoder

BASE = EncoderConfig(vocab_size=200, max_position_embeddings=16, dim=128, n_layers=2, n_heads=2, hidden_dim=256)
RELATIVE = dict(rotary=True, relative_buckets=8, relative_max_distance=6)


def test_the_module_takes_a_plain_encoders_weights_and_nothing_else():
    plain, model = DistilEncoder(BASE), DistilEncoder(dataclasses.replace(BASE, **RELATIVE))
    first = {n: t.clone() for n, t in model.state_dict().items()}
    load_initial_weights(model, plain.state_dict())
    for n, t in model.state_dict().items():
        assert torch.equal(t, plain.state_dict().get(n, first[n])), n
    load_initial_weights(model, first)
    assert all(torch.equal(t, first[n]) for n, t in model.state_dict().items())
    less = dict(plain.state_dict())
    del less["transformer.layer.1.ffn.lin1.weight"]
    for bad in ({}, {"foreign": torch.zeros(1)}, less, {**plain.state_dict(), "foreign": torch.zeros(1)},
                {"encoder." + n: t for n, t in plain.state_dict().items()}):
        with pytest.raises(RuntimeError):
            load_initial_weights(model, bad)
    with pytest.raises(RuntimeError):                # a plain encoder has no place for the new parameters
        load_initial_weights(plain, first)


@pytest.mark.parametrize("options", [["--rotary"], ["--relative-buckets", "8"], []])
def test_the_command_refuses_weights_of_which_nothing_fits(tmp_path, monkeypatch, options):
    import renee_b200.models.encoder as encoder
    monkeypatch.setattr(encoder, "config_from_name", lambda name: BASE)
    torch.save({"foreign": torch.zeros(1)}, tmp_path / "w.pt")
    argv = ["--cpu", "--default-impl", "--synthetic-labels", "40", "--synthetic-train", "16", "--synthetic-test", "8", "--maxlen", "16", "--batch-size", "4",
            "--epochs", "1", "--results-dir", str(tmp_path / "r"), "--encoder-weights", str(tmp_path / "w.pt")] + options
    with pytest.raises(RuntimeError, match="foreign"):
        start(0, 1, build_parser().parse_args(argv))
