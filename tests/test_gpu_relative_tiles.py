"""Relative attention where a CTA takes many tiles, where a row's probabilities leave the range of their reference point, and the 8-bit
GELU where a CTA takes several rounds of rows."""
import dataclasses
import functools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from renee_b200 import ops
from renee_b200.ops.rng import keep_mask
from tests import relative_cases, test_gpu_relative_encoder, test_gpu_relative_ops
from tests.relative_cases import assert_within, attention_inputs, views
from tests.test_gpu_relative_ops import HALF, Attention, dev


def want_on_gpu(monkeypatch, a):
    """attention_64, whose 64-bit products take minutes on the CPU at these sizes."""
    monkeypatch.setattr(relative_cases, "keep_mask", functools.partial(keep_mask, device=dev()))
    with torch.device(dev()):
        want, lim = relative_cases.attention_64({**a.c, **a.g}, a.p, a.rng.seed, a.stream)
    return {n: t.cpu() for n, t in want.items()}, {n: t.cpu() for n, t in lim.items()}


def outputs(a):
    return {n: getattr(a, n).clone() for n in ("ctx", "dq", "dk", "dv", "dtable")}


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_many_tiles_a_cta(hd, p, dt, monkeypatch):
    """1440 tiles on at most 2 CTAs an SM; texts of all lengths with holes, one empty, masked rows full of NaN and infinities."""
    b, S, nh = 40, 300, 12
    assert 3 * b * nh > 4 * 2 * torch.cuda.get_device_properties(0).multi_processor_count
    c = attention_inputs(b, S, nh, hd, dt, "holes", far=40, buckets=16, poison=False)
    c["mask"][b // 2] = 0
    c["mask"][3] = 0
    c["mask"][3, 250] = 1                                # a single key, in the last tile
    c["mask"][5, 70:] = 0                                # tiles without an attended key
    H = nh * hd
    gone = ((c["mask"] == 0) & (c["mask"] != 0).any(1, keepdim=True)).view(-1)
    c["qk"][gone, H:] = float("nan")
    c["qkv"][gone, 2 * H:] = float("inf")
    a = Attention(c, p=p)
    a.fwd()
    a.bwd()
    first = outputs(a)
    want, lim = want_on_gpu(monkeypatch, a)
    for n in want:
        assert_within(n, first[n], want[n], lim[n])
    assert (a.wide[:, 2 * H:3 * H] == 7.0).all()
    for _ in range(2):                                   # tiles go to other CTAs each time
        a.wide.fill_(7.0)
        a.bwd()
        for n, t in outputs(a).items():
            assert torch.equal(t.view(torch.int16), first[n].view(torch.int16)), n
    a.ctx.fill_(7.0)
    a.fwd()
    a.bwd()
    for n, t in outputs(a).items():
        assert torch.equal(t.view(torch.int16), first[n].view(torch.int16)), n


def leaves_its_range(c, up, limit):
    """Of how many rows a piece of 32 keys sums to twice the limit or more beside the largest exponent of the first attended block."""
    b, S, nh, hd = c["b"], c["S"], c["nh"], c["hd"]
    q, k, _ = (t.double().reshape(b, S, nh, hd).transpose(1, 2) for t in views(c))
    far, at = (c["buckets"].numel() - 1) // 2, torch.arange(S)
    bias = c["table"].double()[c["buckets"].long()[(at[None] - at[:, None]).clamp(-far, far) + far]].permute(2, 0, 1)
    s = (q @ k.transpose(-1, -2) / math.sqrt(hd) + bias) / math.log(2.0)
    top = s.abs().max().item()
    s = s.masked_fill((c["mask"] == 0)[:, None, None, :], -math.inf)
    assert (c["mask"][:, :64] != 0).any(1).all()         # the first block has an attended key
    m = s[..., :64].amax(-1, keepdim=True)
    pieces = torch.nn.functional.pad(torch.exp2(s - m + up), (0, -S % 32)).unflatten(-1, (-1, 32)).sum(-1)
    return top, (pieces[..., 2:].amax(-1) > 2 * limit).sum().item()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("kind", ["keys", "table"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_rows_that_leave_the_range_of_their_reference(hd, kind, p, dt):
    """Scores that rise along the sequence, by the keys or by the bias: blocks are worked again, outputs and sums rescaled; the backward
    pass reads what such rows leave."""
    b, S, nh = 2, 400, 2
    rise = 60.0 if dt == torch.bfloat16 else 14.0        # 87 and 20 in base 2: past 2^60 and past 2^15 / 2^6
    c = attention_inputs(b, S, nh, hd, dt, "full", far=320, buckets=64, poison=False)
    g = torch.Generator().manual_seed(2)
    c["mask"] = (torch.rand(b, S, generator=g) > 0.1).int()
    c["mask"][:, :2] = 1
    c["mask"][1, 330:] = 0
    H = nh * hd
    c["qk"] = c["qk"].float() * 0.3
    c["table"] = c["table"].float() * 0.1
    if kind == "keys":
        c["qk"][:, :H] += 8 / math.sqrt(hd)
        c["qk"][:, H:] += (torch.linspace(0, rise / 8, S)[:, None]).repeat(b, 1)
    else:
        c["table"][32:] += torch.linspace(0, rise, 32)[:, None]          # keys behind the query, by their distance
    c["qk"], c["table"] = c["qk"].to(dt), c["table"].to(dt)
    top, rows = leaves_its_range(c, *((0.0, 2.0 ** 60) if dt == torch.bfloat16 else (6.0, 2.0 ** 15)))
    assert rows > 50 and top < 2.0 ** (7 if dt == torch.bfloat16 else 5)
    a = Attention(c, p=p)
    a.fwd()
    a.bwd()
    # attention_64's bounds are for scores of up to 2^5 in base 2, off by 2^-20 of that (2^-15, held to 2^-14).  bf16: up to 2^7, so
    # 2^-13; the bounds are linear in it with other parts beside, so at most twice them
    want, lim = relative_cases.attention_64(c, p, a.rng.seed, a.stream)
    if dt == torch.float16:
        # P~ of keys that few queries look at lies below fp16's normal numbers, where a rounding is off by half of 2^-24; it carries 2^4,
        # the power of two next below sqrt(400), so dv is off by up to 2^-29 of the sum of |dctx| (with P near 2^-20 that is more than u)
        lim["dv"] = lim["dv"] + 2.0 ** -29 * c["dctx"].double().abs().view(b, S, H).sum(1, keepdim=True).expand(b, S, H).reshape(b * S, H)
    for n in want:
        assert_within(n, getattr(a, n), want[n], lim[n] * (2 if dt == torch.bfloat16 else 1))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,F", [(2500, 1536), (1000, 4104)])
def test_gelu8_of_several_rounds(T, F, dt):
    assert T > 32 * (3 * torch.cuda.get_device_properties(0).multi_processor_count // -(-F // 128))
    test_gpu_relative_ops.test_gelu8(T, F, dt)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("change", [dict(), dict(gelu8=False, relative_buckets=0), dict(dim=256, n_heads=8)])
def test_engine_of_long_texts(change, dt):
    test_gpu_relative_encoder.test_engine_tracks_the_oracles(dt, 2, 1100, dict(max_position_embeddings=1100, **change))


def test_training_steps_of_long_texts(monkeypatch):
    monkeypatch.setattr(test_gpu_relative_encoder, "BASE", dataclasses.replace(test_gpu_relative_encoder.BASE, max_position_embeddings=700))
    test_gpu_relative_encoder.test_training_steps_eager_and_captured(700)
