"""Operators of encoder layers with relative positions on the CPU: oracles against 64-bit forms and differences, refusals."""
import math

import pytest
import torch

from renee_b200 import ops
from tests.relative_cases import ATTENTION_SHAPES, assert_within, attention_64, attention_inputs, gelu8_64, rotary_64, shut_behind, views


def run_attention(c, p=0.0, seed=5, stream=3):
    q, k, v = views(c)
    rng = ops.StepRNG(seed)
    ctx, dq, dk, dv = (torch.empty(q.shape, dtype=q.dtype) for _ in range(4))
    dtable = torch.empty_like(c["table"])
    ws = ops.relative_attention_workspace(c["b"], c["S"], c["nh"], c["hd"], 9, q.dtype, "cpu")
    args = (c["mask"], c["table"], c["buckets"], c["nh"], p, rng, stream)
    ops.relative_attention_fwd(q, k, v, *args, ctx, ws)
    ops.relative_attention_bwd(c["dctx"], q, k, v, *args, ctx, ws, dq, dk, dv, dtable)
    return dict(ctx=ctx, dq=dq, dk=dk, dv=dv, dtable=dtable)


@pytest.mark.parametrize("mask", ["full", "padded", "holes", "empty"])
@pytest.mark.parametrize("shape", ATTENTION_SHAPES[:6])
def test_attention_oracle(shape, mask):
    c = attention_inputs(*shape, torch.float32, mask)
    got = run_attention(c, p=0.2)
    want, _ = attention_64(c, 0.2, 5, 3)
    for n, t in want.items():
        torch.testing.assert_close(got[n].double(), t, rtol=2e-4, atol=2e-5)


def test_attention_gradient_of_the_table_by_differences():
    c = attention_inputs(2, 11, 2, 32, torch.float64, "holes", far=4)
    from renee_b200.ops import reference as ref
    q, k, v = views(c)
    got = ref.relative_attention_bwd(c["dctx"], q, k, v, c["mask"], c["table"], c["buckets"], c["nh"], 0.0, 0, 0)[3]

    def loss(table):
        return (ref.relative_attention_fwd(q, k, v, c["mask"], table, c["buckets"], c["nh"], 0.0, 0, 0) * c["dctx"]).sum().item()

    step = 1e-6
    for u in range(c["table"].shape[0]):
        for h in range(2):
            hi, lo = c["table"].clone(), c["table"].clone()
            hi[u, h] += step
            lo[u, h] -= step
            # central differences in 64 bits: step^2 and rounding / step, both far below 1e-6
            assert abs((loss(hi) - loss(lo)) / (2 * step) - got[u, h].item()) < 1e-6


def test_masked_keys_do_not_matter():
    a, b = (attention_inputs(2, 20, 2, 32, torch.float32, "padded", poison=x) for x in (True, False))
    ra, rb = run_attention(a), run_attention(b)
    for n in ra:
        torch.testing.assert_close(ra[n], rb[n], rtol=0, atol=0)


@pytest.mark.parametrize("shut", [float("-inf"), None])
def test_attention_of_distances_that_are_shut(shut):
    """A table entry of minus infinity, or the type's lowest value, takes its distances out."""
    c = shut_behind(attention_inputs(2, 20, 2, 32, torch.float32, "padded", poison=False), shut)
    want, lim = attention_64(c)
    got = run_attention(c)
    for name in want:
        assert_within(name, got[name], want[name], lim[name])
    assert not got["dtable"][4:].any()


def test_buckets():
    far = 128
    b = ops.relative_buckets(32, far).tolist()
    assert len(b) == 2 * far + 1 and b[far] == 0 and set(b) == set(range(32)) - {16}
    assert b[far - 7:far] == [7, 6, 5, 4, 3, 2, 1] and b[far + 1:far + 8] == [17, 18, 19, 20, 21, 22, 23]
    assert [b[far - d] for d in (8, 11, 12, 15, 16, 22, 23, 31, 32, 63, 64, 90, 91, 127, 128)] == \
        [8, 8, 9, 9, 10, 10, 11, 11, 12, 13, 14, 14, 15, 15, 15]
    assert all(x >= y for x, y in zip(b[:far], b[1:far]))
    for bad in ((3, 128), (5, 128), (32, 8), (32, 2000)):
        with pytest.raises(ValueError):
            ops.relative_buckets(*bad)


@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("b,S,nh,hd", [(1, 1, 1, 32), (3, 7, 2, 64), (2, 5, 3, 128), (0, 4, 2, 32)])
def test_rotary_oracle(b, S, nh, hd, with_positions):
    g = torch.Generator().manual_seed(1)
    T = b * S
    x, dy = (torch.randn(T, 2 * nh * hd, generator=g) for _ in range(2))
    gq, gk = (torch.randn(hd, generator=g) for _ in range(2))
    table = ops.rotary_table(50, hd)
    pos = torch.randint(0, 50, (T,), generator=g, dtype=torch.int32) if with_positions else None
    y, dx, dgq, dgk = torch.empty_like(x), torch.empty_like(x), torch.empty_like(gq), torch.empty_like(gk)
    ops.qk_norm_rotary_fwd(x, gq, gk, table, S, nh, 1e-6, y, positions=pos)
    ops.qk_norm_rotary_bwd(dy, x, gq, gk, table, S, nh, 1e-6, ops.qk_norm_rotary_workspace(T, nh, hd, "cpu"), dx, dgq, dgk, positions=pos)
    at = pos.long() if with_positions else torch.arange(T) % S
    for got, want in zip((y, dx, dgq, dgk), rotary_64(x, gq, gk, table, at, nh, 1e-6, dy)):
        torch.testing.assert_close(got.double(), want, rtol=1e-4, atol=1e-5)


def test_rotary_table_of_a_far_position():
    t = ops.rotary_table(100001, 64)
    i = 3
    angle = 100000 * 10000.0 ** (-i / 32)
    assert abs(t[100000, i].item() - math.cos(angle)) < 1e-7 and abs(t[100000, 32 + i].item() - math.sin(angle)) < 1e-7


def test_rotary_products_depend_on_distance_alone():
    hd, S = 32, 12
    x = torch.randn(1, 2 * hd, generator=torch.Generator().manual_seed(2)).repeat(S, 1)
    y = torch.empty_like(x)
    one = torch.ones(hd)
    ops.qk_norm_rotary_fwd(x, one, one, ops.rotary_table(S, hd), S, 1, 1e-6, y)
    s = y[:, :hd] @ y[:, hd:].T
    for d in range(-S + 1, S):
        line = torch.diagonal(s, d)
        torch.testing.assert_close(line, line[:1].expand_as(line), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("T,F", [(1, 8), (5, 128), (4, 200), (3, 512)])
def test_gelu8_oracle(T, F):
    g = torch.Generator().manual_seed(3)
    x, da = (torch.randn(T, F, generator=g) * 3 for _ in range(2))
    bias = torch.randn(F, generator=g)
    saved = ops.gelu8_saved(T, F, "cpu")
    out, dx, act, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty(F)
    ops.gelu8_fwd(x, bias, out, saved)
    ops.gelu8_bwd(da, saved, ops.gelu8_workspace(T, F, "cpu"), db, dx, act)
    want_out, held, want_dx, want_act, want_db = gelu8_64(x, bias, da)
    for got, want in ((out, want_out), (dx, want_dx), (act, want_act), (db, want_db)):
        torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)
    z = x.double() + bias.double()
    for at in range(0, F, 128):                      # half a step of the block, and the fp32 rounding of the scale
        top = z[:, at:at + 128].abs().amax(1, keepdim=True)
        assert ((held - z)[:, at:at + 128].abs() <= top / 254 * (1 + 1e-6)).all()


def test_gelu8_edges():
    x = torch.zeros(4, 128)
    x[1, 5], x[2, 7], x[3, 9] = float("inf"), float("nan"), 1e-35
    saved = ops.gelu8_saved(4, 128, "cpu")
    out = torch.empty_like(x)
    ops.gelu8_fwd(x, torch.zeros(128), out, saved)
    assert torch.isnan(saved.scale[1:3]).all() and (saved.scale[[0, 3]] == 0).all() and (saved.q == 0).all()


def _attention_call(**change):
    c = attention_inputs(2, 8, 2, 32, torch.float32)
    q, k, v = views(c)
    a = dict(q=q, k=k, v=v, mask=c["mask"], table=c["table"], buckets=c["buckets"], nh=2, p=0.0, rng=None, stream=0, ctx_out=torch.empty(16, 64),
             ws=ops.relative_attention_workspace(2, 8, 2, 32, 9, torch.float32, "cpu"))
    a.update(change)
    ops.relative_attention_fwd(**a)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(16, 60)), dict(q=torch.zeros(15, 64)), dict(nh=3), dict(nh=0), dict(k=torch.zeros(16, 64, dtype=torch.bfloat16)),
    dict(v=torch.zeros(64, 16).t()), dict(mask=torch.ones(2, 8)), dict(mask=torch.ones(2, 0, dtype=torch.int32)), dict(mask=torch.ones(16, dtype=torch.int32)),
    dict(table=torch.zeros(8, 3)), dict(table=torch.zeros(0, 2)), dict(buckets=torch.zeros(4, dtype=torch.int32)), dict(buckets=torch.zeros(9)),
    dict(buckets=torch.zeros(5001, dtype=torch.int32)), dict(p=1.0), dict(p=0.995), dict(p=-0.1), dict(p=0.5), dict(ctx_out=torch.zeros(16, 128)[:, :64]),
    dict(q=torch.zeros(16 * 64 + 1)[1:].view(16, 64)), dict(q=torch.zeros(16 * 66).as_strided((16, 64), (66, 1)))])
def test_attention_refuses(change):
    with pytest.raises(ValueError):
        _attention_call(**change)


def test_attention_refuses_shared_memory():
    x = torch.zeros(16, 64)
    with pytest.raises(ValueError, match="same memory"):
        _attention_call(q=x, ctx_out=x)


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(6, 100)), dict(x=torch.zeros(6, 128, dtype=torch.float64)), dict(gq=torch.zeros(16)), dict(S=4), dict(S=0), dict(nh=0),
    dict(table=torch.zeros(2, 32)), dict(table=torch.zeros(9, 16)), dict(table=torch.zeros(9, 32).double()), dict(eps=0.0),
    dict(positions=torch.zeros(5, dtype=torch.int32)), dict(positions=torch.zeros(6)), dict(out=torch.zeros(6, 64))])
def test_rotary_refuses(change):
    a = dict(x=torch.zeros(6, 128), gq=torch.zeros(32), gk=torch.zeros(32), table=torch.zeros(9, 32), S=3, nh=2, eps=1e-6, out=torch.zeros(6, 128))
    ops.qk_norm_rotary_fwd(**a)
    a.update(change)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary_fwd(**a)


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(4, 12)), dict(x=torch.zeros(4, 16).double()), dict(bias=torch.zeros(8)), dict(out=torch.zeros(4, 32)[:, :16]),
    dict(saved=ops.gelu8_saved(4, 8, "cpu")), dict(saved=ops.gelu8_saved(5, 16, "cpu"))])
def test_gelu8_refuses(change):
    a = dict(x=torch.zeros(4, 16), bias=torch.zeros(16), out=torch.zeros(4, 16), saved=ops.gelu8_saved(4, 16, "cpu"))
    ops.gelu8_fwd(**a)
    a.update(change)
    with pytest.raises(ValueError):
        ops.gelu8_fwd(**a)


@pytest.mark.parametrize("heads", [0, 1, 5, 7])
def test_dropout_numbers_beyond_32_bits(heads, monkeypatch):
    """Heads that share a stream are numbered through; no two heads share their decisions, however many there are."""
    from renee_b200.ops.rng import PairNumbers, keep_mask
    S, p = 40, 0.4
    assert torch.equal(PairNumbers(3, S).keep_mask(5, heads, p), keep_mask(5, 3, (heads, S, S), p))
    monkeypatch.setattr(PairNumbers, "NUMBERS", 2 * S * S + 17)                    # two heads a stream
    n = PairNumbers(3, S)
    assert n.page == 2 and [n.of(h) for h in range(5)] == [(3, 0), (3, S * S), (4099, 0), (4099, S * S), (8195, 0)]
    got = n.keep_mask(5, heads, p)
    assert got.shape == (heads, S, S)
    for h in range(heads):
        stream, first = n.of(h)
        assert torch.equal(got[h].reshape(-1), keep_mask(5, stream, (first + S * S,), p)[first:])
        for other in range(h):                       # independent decisions agree at p^2 + (1 - p)^2 = 0.52 of 1600 places: 6 deviations
            assert abs((got[h] == got[other]).float().mean().item() - 0.52) < 6 * 0.0125


def test_dropout_numbers_of_the_longest_sequences():
    from renee_b200.ops.rng import PairNumbers
    n = PairNumbers(12, 65536)
    assert n.page == 1 and [n.of(h) for h in (0, 1, 70000)] == [(12, 0), (12 + 4096, 0), (12 + 4096 * 70000, 0)]


def test_attention_oracle_takes_heads_beyond_32_bits(monkeypatch):
    from renee_b200.ops import reference as ref
    from renee_b200.ops.rng import PairNumbers
    b, S, nh, hd = 3, 10, 2, 32
    monkeypatch.setattr(PairNumbers, "NUMBERS", 4 * S * S)
    T, H = b * S, nh * hd
    zero, v = torch.zeros(T, H), torch.randn(T, H, generator=torch.Generator().manual_seed(0))
    args = (torch.ones(b, S, dtype=torch.int32), torch.zeros(8, nh), ops.relative_buckets(8, 4), nh, 0.5, 7, 3)
    w = PairNumbers(3, S).keep_mask(7, b * nh, 0.5).view(b, nh, S, S).float() * 2 / S
    heads = lambda t: t.view(b, S, nh, hd).transpose(1, 2)
    got = ref.relative_attention_fwd(zero, zero, v, *args)
    torch.testing.assert_close(heads(got), w @ heads(v))
    dv = ref.relative_attention_bwd(v, zero, zero, v, *args)[2]
    torch.testing.assert_close(heads(dv), w.transpose(-1, -2) @ heads(v))
