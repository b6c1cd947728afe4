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


def test_the_engine_refuses_an_encoder_of_another_kind():
    plain, rel = FlatEncoder(BASE, "cpu", torch.float32), FlatEncoder(dataclasses.replace(BASE, **RELATIVE), "cpu", torch.float32)
    rel.load_encoder_state_dict(plain.encoder_state_dict())
    with pytest.raises(KeyError, match="relative"):
        plain.load_encoder_state_dict(rel.encoder_state_dict())
    with pytest.raises(KeyError, match="missing"):
        rel.load_encoder_state_dict(plain.encoder_state_dict(), initial=False)
    rel.load_encoder_state_dict(rel.encoder_state_dict(), initial=False)


def test_a_trained_state_is_not_taken_by_an_encoder_of_another_kind():
    from renee_b200.parallel.dist import DistContext
    from renee_b200.train import TrainConfig, XCTrainer
    from renee_b200.utils.sharding import shard_labels
    cfg = TrainConfig(batch_size=4, epochs=1, seed=0, dropout=0.3, lr1=0.05, lr2=1e-3, warmup=2, wd1=1e-4, noloss=True, maxlen=8, pooling="mean")
    plain, rel = (XCTrainer(cfg, c, shard_labels(40, 1), DistContext(device=torch.device("cpu")), steps_per_epoch=2)
                  for c in (BASE, dataclasses.replace(BASE, **RELATIVE)))
    for tr, other in ((plain, rel), (rel, plain)):
        with pytest.raises(KeyError):
            tr.load_state_dict(other.state_dict())
        tr.load_state_dict(tr.state_dict())


@pytest.mark.parametrize("buckets,far", [(-4, 128), (3, 128), (32, 8), (32, 513), (32, 0)])
def test_encoders_refuse_buckets_that_there_are_not(buckets, far):
    with pytest.raises(ValueError, match="no buckets"):
        dataclasses.replace(BASE, relative_buckets=buckets, relative_max_distance=far)
    assert dataclasses.replace(BASE, relative_max_distance=far).relative_buckets == 0


@pytest.mark.parametrize("options", [["--relative-buckets", "-4"], ["--relative-buckets", "32", "--relative-max-distance", "600"],
                                     ["--default-impl", "--gelu8"]])
def test_the_command_refuses_options_that_it_cannot_follow(tmp_path, monkeypatch, options):
    import renee_b200.models.encoder as encoder
    monkeypatch.setattr(encoder, "config_from_name", lambda name: BASE)
    argv = ["--cpu", "--synthetic-labels", "40", "--synthetic-train", "16", "--synthetic-test", "8", "--maxlen", "16", "--batch-size", "4",
            "--epochs", "1", "--results-dir", str(tmp_path / "r")] + options
    with pytest.raises(ValueError, match="no buckets|engine"):
        start(0, 1, build_parser().parse_args(argv))
