"""Gradients of the relative attention beyond fp16's range: dS, an operand in 16 bits, may be larger than what comes of it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from renee_b200 import ops
from tests.relative_cases import assert_within, attention_64, attention_inputs, views
from tests.test_gpu_relative_ops import Attention
from tests.test_gpu_relative_tiles import outputs, want_on_gpu

SHAPES = [(2, 20, 3, 32), (3, 16, 2, 64), (2, 50, 2, 64), (2, 64, 1, 128), (3, 65, 2, 64), (2, 300, 3, 64), (1, 517, 2, 32), (2, 129, 2, 128)]


def large_inputs(shape, rows, mask="holes", dt=torch.float16):
    """Small queries and keys, large values and gradients: of all rows or of a few of each sequence."""
    c = attention_inputs(*shape, dt, mask, poison=False)
    b, S, nh, hd = shape
    H = nh * hd
    c["qk"] = (c["qk"].float() * 0.015).to(dt)
    c["qkv"] = (c["qkv"].float() * 100).to(dt)
    size = torch.ones(b, S, 1)
    size[:, :: 1 if rows == "all" else 11] = 6000
    c["dctx"] = (c["dctx"].float().view(b, S, H) * size).view(b * S, H).to(dt)
    gone = ((c["mask"] == 0) & (c["mask"] != 0).any(1, keepdim=True)).view(-1)
    c["qk"][gone, H:] = float("nan")
    c["qkv"][gone, 2 * H:] = float("inf")
    return c


def largest(c, p):
    """(the largest |dS| there can be in each sequence and head, the largest there is)"""
    b, S, nh, hd = c["b"], c["S"], c["nh"], c["hd"]
    heads = lambda t: t.double().reshape(b, S, nh, hd).transpose(1, 2)
    q, k, v = (heads(t) for t in views(c))
    use = (c["mask"] != 0) | (c["mask"] == 0).all(1, keepdim=True)
    k, v = (torch.where(use[:, None, :, None], t, torch.zeros_like(t)) for t in (k, v))
    do = heads(c["dctx"])
    most = 2 * do.norm(dim=-1).amax(-1) * v.norm(dim=-1).amax(-1) / (1 - p)
    far, at = (c["buckets"].numel() - 1) // 2, torch.arange(S)
    s = q @ k.transpose(-1, -2) / math.sqrt(hd) + c["table"].double()[c["buckets"].long()[(at[None] - at[:, None]).clamp(-far, far) + far]].permute(2, 0, 1)
    w = torch.softmax(s.masked_fill(~use[:, None, None, :], -math.inf), -1)
    dp = do @ v.transpose(-1, -2)
    return most, (w * (dp - (w * dp).sum(-1, keepdim=True))).abs().max().item()


def widen(lim, c, most):
    """The factor takes the largest dS there can be to 2^14 or beyond, where fp16's least step, 2^-24, is 2^-38 of it: off by half of that."""
    b, S, nh, hd = c["b"], c["S"], c["nh"], c["hd"]
    rows_of = lambda t: t.transpose(1, 2).reshape(b * S, nh * hd)
    heads = lambda t: t.double().reshape(b, S, nh, hd).transpose(1, 2)
    q, k, _ = (heads(t) for t in views(c))
    use = (c["mask"] != 0) | (c["mask"] == 0).all(1, keepdim=True)
    k = torch.where(use[:, None, :, None], k, torch.zeros_like(k))
    step = (most * 2.0 ** -39 / math.sqrt(hd))[:, :, None, None]
    lim["dq"] = lim["dq"] + rows_of((step * k.abs().sum(2, keepdim=True)).expand(b, nh, S, hd))
    lim["dk"] = lim["dk"] + rows_of((step * q.abs().sum(2, keepdim=True)).expand(b, nh, S, hd))
    lim["dtable"] = lim["dtable"] + (most * 2.0 ** -39).sum(0) * S * S
    return lim


def check_table(got, want, lim):
    """Entries beyond the type are infinite, as they are when the exact ones are rounded."""
    got, over, fits = got.double().cpu(), want.abs() > 65520 + lim, want.abs() < 65504 - lim
    assert torch.equal(got[over], torch.sign(want[over]) * math.inf)
    assert_within("dtable", got[fits], want[fits], lim[fits])


@pytest.mark.parametrize("rows", ["all", "few"])
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("shape", SHAPES)
def test_large_gradients(shape, p, rows):
    b, S, nh, hd = shape
    c = large_inputs(shape, rows)
    most, there_is = largest(c, p)
    assert there_is > 65504                              # of what the factor in front leaves room for less: 65504 / sqrt(S)
    a = Attention(c, p=p)
    a.fwd()
    a.bwd()
    want, lim = attention_64(c, p, a.rng.seed, a.stream)
    assert all(want[n].abs().max() < 60000 for n in ("ctx", "dq", "dk", "dv"))
    lim = widen(lim, c, most)
    for n in ("ctx", "dq", "dk", "dv"):
        assert_within(n, getattr(a, n), want[n], lim[n])
    check_table(a.dtable, want["dtable"], lim["dtable"])
    H = nh * hd
    assert (a.wide[:, 2 * H:3 * H] == 7.0).all()


@pytest.mark.parametrize("shape", [(3, 40, 2, 64), (3, 200, 2, 64), (3, 150, 1, 128)])
def test_a_gradient_that_is_not_finite_stays_where_it_is(shape):
    """An infinity in one row of one head of dctx: other rows of dq, other sequences and heads have what they had."""
    b, S, nh, hd = shape
    c = attention_inputs(*shape, torch.float16, "full", poison=False)
    clean = Attention(c)
    dirty = Attention(dict(c, dctx=c["dctx"].clone()))
    dirty.g["dctx"][S + 7, 3] = float("inf")
    for a in (clean, dirty):
        a.fwd()
        a.bwd()
    clean.check()
    rows = torch.arange(b * S, device="cuda:0") == S + 7
    assert not torch.isfinite(dirty.dq[rows][:, :hd]).any()
    assert torch.equal(dirty.dq[~rows], clean.dq[~rows]) and torch.equal(dirty.dq[rows][:, hd:], clean.dq[rows][:, hd:])
    for n in ("dk", "dv"):
        x, y = getattr(dirty, n), getattr(clean, n)
        other = torch.arange(b * S, device="cuda:0") // S != 1
        assert torch.equal(x[other], y[other]) and torch.equal(x[:, hd:], y[:, hd:])


@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_tiles_of_both_kinds(hd, p, monkeypatch):
    """Large gradients in some heads of some sequences, 1440 tiles on at most 2 CTAs an SM, some without an attended key."""
    b, S, nh = 40, 300, 12
    c = large_inputs((b, S, nh, hd), "few")
    large = (torch.arange(b)[:, None] % 3 == 0) & (torch.arange(nh)[None] % 4 != 1)
    c["dctx"] = torch.where(large[:, None, :, None], c["dctx"].view(b, S, nh, hd), c["dctx"].view(b, S, nh, hd) / 240000).reshape(b * S, nh * hd)
    most, there_is = largest(c, p)
    assert there_is > 65504 and most[~large].max() < 2.0 ** 11 and most[large].min() > 2.0 ** 22
    a = Attention(c, p=p)
    a.fwd()
    a.bwd()
    first = outputs(a)
    want, lim = want_on_gpu(monkeypatch, a)
    lim = widen(lim, c, most)
    for n in ("ctx", "dq", "dk", "dv"):
        assert_within(n, first[n], want[n], lim[n])
    check_table(first["dtable"], want["dtable"], lim["dtable"])
    for _ in range(2):
        a.wide.fill_(7.0)
        a.bwd()
        for n, t in outputs(a).items():
            assert torch.equal(t.view(torch.int16), first[n].view(torch.int16)), n
    # the same heads as before once the large ones are gone
    c["dctx"] = torch.where(large[:, None, :, None], torch.zeros(()).half(), c["dctx"].view(b, S, nh, hd)).reshape(b * S, nh * hd)
    quiet = Attention(c, p=p)
    quiet.fwd()
    quiet.bwd()
    kept = (~large)[:, None, :, None].expand(b, S, nh, hd).reshape(b * S, nh * hd)
    for n in ("dq", "dk", "dv"):
        assert torch.equal(getattr(quiet, n).cpu()[kept], first[n].cpu()[kept]), n
