"""Encoders with relative positions and 8-bit pre-activations: the engine's forward and backward passes against autograd."""
import dataclasses

import pytest
import torch

from renee_b200 import ops
from renee_b200.cli import _encoder_config, build_parser
from renee_b200.models.encoder import DistilEncoder, EncoderConfig, TransformerInputLayer
from renee_b200.models.flat_encoder import FlatEncoder

BASE = EncoderConfig(vocab_size=200, max_position_embeddings=16, dim=128, n_layers=2, n_heads=2, hidden_dim=256, dropout=0.0, attention_dropout=0.0)
VARIANTS = {"rotary": dict(rotary=True), "relative": dict(relative_buckets=8, relative_max_distance=6),
            "both": dict(rotary=True, relative_buckets=8, relative_max_distance=6)}


def inputs(b=5, S=12):
    g = torch.Generator().manual_seed(0)
    mask = (torch.arange(S)[None] < torch.randint(3, S + 1, (b, 1), generator=g)).int()
    return torch.randint(1, 200, (b, S), generator=g).int() * mask, mask


def pair(cfg, pooling="mean"):
    torch.manual_seed(1)
    mod = DistilEncoder(cfg).double()
    with torch.no_grad():
        for n, p in mod.named_parameters():
            if "bias" in n or "norm" in n.lower():
                p.add_(0.1 * torch.randn_like(p))
    flat = FlatEncoder(cfg, "cpu", torch.float32, pooling, seed=3)
    flat.load_encoder_state_dict({k: v.float() for k, v in mod.state_dict().items()})
    return mod, TransformerInputLayer(mod, pooling), flat


def compare_gradients(mod, flat, pad):
    for n, p in mod.named_parameters():
        want = p.grad.float()
        if n == "embeddings.word_embeddings.weight":
            want = want.clone()
            want[pad] = 0
        torch.testing.assert_close(flat.view(flat.g, n), want, rtol=2e-3, atol=2e-5, msg=lambda m: f"{n}: {m}")


@pytest.mark.parametrize("empty", [False, True])
@pytest.mark.parametrize("variant", sorted(VARIANTS))
def test_engine_matches_autograd(variant, empty):
    cfg = dataclasses.replace(BASE, **VARIANTS[variant])
    mod, wrap, flat = pair(cfg, "cls" if empty else "mean")
    assert set(flat.encoder_state_dict()) == set(mod.state_dict())
    ids, mask = inputs()
    if empty:
        mask[2] = 0                                  # nothing is attended: uniform over all tokens, as in the module
    e_ref = wrap({"input_ids": ids, "attention_mask": mask})
    e = flat.forward(ids, mask, ops.StepRNG(0), train=True)
    torch.testing.assert_close(e.double(), e_ref.double(), rtol=2e-4, atol=2e-5)
    d = torch.randn(e.shape, generator=torch.Generator().manual_seed(5))
    e_ref.backward(d.double())
    flat.backward(d.clone())
    compare_gradients(mod, flat, cfg.pad_token_id)
    if "relative_buckets" in VARIANTS[variant]:
        assert flat.view(flat.g, "transformer.layer.1.attention.relative_bias.weight").abs().max() > 0


class Held(torch.autograd.Function):
    """GELU and the linear behind it, differentiated from a pre-activation held in 8 bits."""

    @staticmethod
    def forward(ctx, z, w, b):
        held = torch.empty_like(z)
        for at in range(0, z.shape[-1], 128):
            part = z[..., at:at + 128]
            unit = part.abs().amax(-1, keepdim=True) / 127
            held[..., at:at + 128] = torch.round(part / unit) * unit
        ctx.save_for_backward(held, w)
        return torch.nn.functional.gelu(z) @ w.t() + b

    @staticmethod
    def backward(ctx, dy):
        held, w = ctx.saved_tensors
        with torch.enable_grad():
            h = held.detach().requires_grad_()
            a = torch.nn.functional.gelu(h)
        (dz,) = torch.autograd.grad(a, h, dy @ w)
        rows = dy.reshape(-1, dy.shape[-1])
        return dz, rows.t() @ a.detach().reshape(-1, a.shape[-1]), rows.sum(0)


def test_engine_with_8_bit_pre_activations():
    cfg = dataclasses.replace(BASE, gelu8=True, **VARIANTS["both"])
    mod, wrap, flat = pair(cfg)
    for blk in mod.transformer.layer:
        blk.ffn.forward = lambda x, f=blk.ffn: Held.apply(f.lin1(x), f.lin2.weight, f.lin2.bias)
    plain = FlatEncoder(dataclasses.replace(cfg, gelu8=False), "cpu", torch.float32, "mean", seed=3)
    plain.load_encoder_state_dict(flat.encoder_state_dict())
    ids, mask = inputs()
    e_ref = wrap({"input_ids": ids, "attention_mask": mask})
    e = flat.forward(ids, mask, ops.StepRNG(0), train=True)
    assert torch.equal(e, plain.forward(ids, mask, ops.StepRNG(0), train=True))       # the forward pass is not changed
    d = torch.randn(e.shape, generator=torch.Generator().manual_seed(5))
    e_ref.backward(d.double())
    flat.backward(d.clone())
    compare_gradients(mod, flat, cfg.pad_token_id)
    assert flat._acts["layers"][0]["f1"] is flat._acts["layers"][1]["f1"]             # one 16-bit pre-activation for all layers


def test_layout_of_the_new_parameters():
    flat = FlatEncoder(dataclasses.replace(BASE, **VARIANTS["both"]), "cpu", torch.float32)
    matrices = [s.offset for n, s in flat.slots.items() if len(s.shape) == 2 and "relative_bias" not in n]
    for l in range(2):
        p = f"transformer.layer.{l}.attention."
        assert max(matrices) < flat.slots[p + "q_norm.weight"].offset < flat.n_decay       # behind the matrices, decayed as the block norms
        assert flat.slots[p + "relative_bias.weight"].offset >= flat.n_decay
        assert (flat.view(flat.p32, p + "q_norm.weight") == 1).all()


def test_weights_without_relative_positions_can_be_loaded():
    old = FlatEncoder(BASE, "cpu", torch.float32, seed=1)
    new = FlatEncoder(dataclasses.replace(BASE, **VARIANTS["both"]), "cpu", torch.float32, seed=2)
    new.load_encoder_state_dict(old.encoder_state_dict())
    n = "transformer.layer.1.ffn.lin1.weight"
    assert torch.equal(new.view(new.p32, n), old.view(old.p32, n))
    with pytest.raises(KeyError):
        new.load_encoder_state_dict({})


def test_weights_with_fewer_positions_can_be_loaded():
    from renee_b200.models.encoder import grow_positions
    n = "embeddings.position_embeddings.weight"
    longer = dataclasses.replace(BASE, **VARIANTS["both"], max_position_embeddings=BASE.max_position_embeddings + 9)
    old, new = FlatEncoder(BASE, "cpu", torch.float32, seed=1), FlatEncoder(longer, "cpu", torch.float32, seed=2)
    own = new.view(new.p32, n).clone()
    new.load_encoder_state_dict(grow_positions(old.encoder_state_dict(), own))
    assert torch.equal(new.view(new.p32, n), torch.cat([old.view(old.p32, n), own[-9:]]))
    model = DistilEncoder(longer)
    model.load_state_dict(grow_positions(old.encoder_state_dict(), model.state_dict()[n]), strict=False)
    assert torch.equal(model.state_dict()[n][:-9], old.view(old.p32, n))


def test_command_line():
    parse = build_parser().parse_args
    assert _encoder_config(parse([])) == EncoderConfig()
    cfg = _encoder_config(parse(["--rotary", "--relative-buckets", "32", "--gelu8", "--maxlen", "1024"]))
    assert cfg.rotary and cfg.relative_buckets == 32 and cfg.relative_max_distance == 128 and cfg.gelu8 and cfg.max_position_embeddings == 1024
    assert _encoder_config(parse(["--maxlen", "1024"])).max_position_embeddings == 512


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_the_module_rotates_by_cosines_in_32_bits(dt, monkeypatch):
    from renee_b200.ops import reference
    seen = []
    whole = reference.qk_norm_rotary_fwd
    monkeypatch.setattr(reference, "qk_norm_rotary_fwd", lambda *a: seen.append(a[3]) or whole(*a))
    mod = DistilEncoder(dataclasses.replace(BASE, rotary=True)).to(dt)
    ids, mask = inputs()
    mod(input_ids=ids, attention_mask=mask)
    assert len(seen) == 2 and all(torch.equal(t, ops.rotary_table(12, 64)) for t in seen)


@pytest.mark.parametrize("change", [dict(), *VARIANTS.values()])
def test_longer_texts_than_positions_are_refused(change):
    """The table of learned positions has a row for each: there is none to read, nor to write a gradient to, behind the last."""
    flat = FlatEncoder(dataclasses.replace(BASE, **change), "cpu", torch.float32)
    ids, mask = inputs(S=BASE.max_position_embeddings)
    flat.forward(ids, mask, ops.StepRNG(0), train=True)
    with pytest.raises(ValueError, match="17 tokens"):
        flat.forward(*(torch.cat([t, t[:, :1]], 1) for t in (ids, mask)), ops.StepRNG(0), train=True)
