"""Kernels of the operators of encoder layers with relative positions against plain 64-bit forms (tests/relative_cases.py, which
derives the bounds of the attention's 16-bit operands)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from renee_b200 import ops
from tests.relative_cases import (ATTENTION_SHAPES, assert_within, attention_64, attention_inputs, gelu8_64, rotary_64, shut_behind, u_of, views)

HALF = [torch.bfloat16, torch.float16]


def dev():
    return torch.device("cuda", 0)


class Attention:
    """The buffers of one call, as views with guard columns of a wider matrix."""

    def __init__(self, c, p=0.0, seed=5, stream=3):
        self.c, self.p, self.stream = c, p, stream
        g = {n: t.to(dev()) if torch.is_tensor(t) else t for n, t in c.items()}
        self.g = g
        H, T = c["nh"] * c["hd"], c["b"] * c["S"]
        self.q, self.k, self.v = g["qk"][:, :H], g["qk"][:, H:], g["qkv"][:, 2 * H:]
        self.rng = ops.StepRNG(seed, torch.tensor([seed], dtype=torch.int32, device=dev()))
        self.ctx = torch.full((T, H), 7.0, dtype=c["qk"].dtype, device=dev())
        self.wide = torch.full((T, 4 * H), 7.0, dtype=c["qk"].dtype, device=dev())
        self.dq, self.dk, self.dv = self.wide[:, :H], self.wide[:, H:2 * H], self.wide[:, 3 * H:]
        self.dtable = torch.full_like(g["table"], 7.0)
        self.ws = ops.relative_attention_workspace(c["b"], c["S"], c["nh"], c["hd"], (c["buckets"].numel() - 1) // 2, c["qk"].dtype, dev())

    def args(self):
        return (self.g["mask"], self.g["table"], self.g["buckets"], self.c["nh"], self.p, self.rng, self.stream)

    def fwd(self):
        ops.relative_attention_fwd(self.q, self.k, self.v, *self.args(), self.ctx, self.ws)

    def bwd(self):
        ops.relative_attention_bwd(self.g["dctx"], self.q, self.k, self.v, *self.args(), self.ctx, self.ws, self.dq, self.dk, self.dv, self.dtable)

    def check(self):
        want, lim = attention_64(self.c, self.p, self.rng.seed, self.stream)
        for n in want:
            assert_within(n, getattr(self, n), want[n], lim[n])
        H = self.c["nh"] * self.c["hd"]
        assert (self.wide[:, 2 * H:3 * H] == 7.0).all()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("mask", ["full", "holes", "empty"])
@pytest.mark.parametrize("shape", ATTENTION_SHAPES)
def test_attention(shape, mask, dt):
    a = Attention(attention_inputs(*shape, dt, mask))
    a.fwd()
    a.bwd()
    a.check()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("shape", [(3, 7, 2, 32), (2, 33, 2, 64), (2, 129, 2, 128), (2, 300, 3, 64)])
def test_attention_dropout(shape, dt):
    a = Attention(attention_inputs(*shape, dt, "padded"), p=0.3)
    a.fwd()
    a.bwd()
    a.check()


@pytest.mark.parametrize("far,buckets,S", [(3, 4, 40), (128, 32, 40), (128, 32, 300), (512, 64, 200), (512, 64, 700), (40, 16, 600)])
def test_attention_windows(far, buckets, S):
    """Bucket maps shorter and longer than the sequence and than a tile."""
    a = Attention(attention_inputs(2, S, 2, 64, torch.bfloat16, "padded", far=far, buckets=buckets))
    a.fwd()
    a.bwd()
    a.check()


def test_attention_map_in_any_order():
    c = attention_inputs(2, 150, 2, 64, torch.bfloat16, "padded", far=20, buckets=8)
    c["buckets"] = torch.randint(0, 8, (41,), generator=torch.Generator().manual_seed(9), dtype=torch.int32)
    a = Attention(c)
    a.fwd()
    a.bwd()
    a.check()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("S", [1, 20, 64, 150])
def test_attention_of_single_keys_has_no_gradient_but_of_v(S, p, dt):
    """One attended key: P is 1 whatever the scores are, so their gradients are zeros, not rounding."""
    c = attention_inputs(5, S, 2, 64, dt, "full", poison=False)
    c["mask"][:] = 0
    for i in range(5):
        c["mask"][i, (i * 37) % S] = 1
    a = Attention(c, p=p)
    a.fwd()
    a.bwd()
    a.check()
    assert not a.dq.any() and not a.dk.any() and not a.dtable.any()


def test_attention_far_scores():
    """Scores up to about 300 in base e: the running maximum moves from block to block."""
    c = attention_inputs(1, 260, 2, 64, torch.bfloat16, "full", poison=False)
    ramp = torch.linspace(0.2, 6.0, 260)[:, None]
    c["qk"] = (c["qk"].float() * ramp).bfloat16()
    a = Attention(c)
    a.fwd()
    want, _ = attention_64(c)
    # P off by the scores' fp32 rounding: 2^-22 of sums of magnitudes up to 400 log2 e; as an operand by 2^-9; ctx by 2^-9
    torch.testing.assert_close(a.ctx.double().cpu(), want["ctx"], rtol=2.0 ** -7, atol=2.0 ** -8 * 4)


@pytest.mark.parametrize("S", [33, 200])
def test_attention_of_an_empty_sequence_reads_no_scores(S):
    """Where nothing is attended, q and k do not matter, NaNs included, and have no gradient."""
    c = attention_inputs(3, S, 2, 64, torch.bfloat16, "empty", poison=False)
    clean = Attention(c)
    nans = c["qk"].clone()
    nans[S:2 * S] = float("nan")
    dirty = Attention(dict(c, qk=nans))
    for a in (clean, dirty):
        a.fwd()
        a.bwd()
    clean.check()
    assert torch.equal(clean.ctx, dirty.ctx) and torch.equal(clean.wide, dirty.wide) and torch.equal(clean.dtable, dirty.dtable)
    assert not dirty.dq[S:2 * S].any() and not dirty.dk[S:2 * S].any()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("shut", [float("-inf"), None])
@pytest.mark.parametrize("S,far", [(20, 9), (60, 9), (200, 9), (300, 128)])
def test_attention_of_distances_that_are_shut(S, far, shut, dt):
    a = Attention(shut_behind(attention_inputs(2, S, 2, 64, dt, "padded", far=far, poison=False), shut))
    a.fwd()
    a.bwd()
    a.check()
    assert not a.dtable[4:].any()


@pytest.mark.parametrize("S", [30, 64, 70, 129, 200])
def test_attention_in_a_larger_workspace_and_backward_again(S):
    """A workspace for more sequences of more tokens, used for larger and smaller calls in turn; each backward pass runs twice."""
    ws = ops.relative_attention_workspace(5, 200, 2, 64, 9, torch.bfloat16, dev())
    for b, s in ((5, 200), (2, S), (5, 200), (1, S)):
        a = Attention(attention_inputs(b, s, 2, 64, torch.bfloat16, "holes"))
        a.ws = ws
        a.fwd()
        for _ in range(2):
            a.wide.fill_(7.0)
            a.dtable.fill_(7.0)
            a.bwd()
            a.check()


@pytest.mark.parametrize("shape", [(2, 20, 2, 64), (3, 70, 2, 64), (2, 129, 3, 32), (2, 200, 1, 128)])
def test_attention_leaves_what_lies_behind(shape):
    """Outputs as the first rows of longer matrices."""
    a = Attention(attention_inputs(*shape, torch.bfloat16, "padded"))
    T, H = a.ctx.shape
    more = [torch.full((T + 130, w), 7.0, dtype=torch.bfloat16, device=dev()) for w in (H, 4 * H)]
    a.ctx, a.wide = (m[:T] for m in more)
    a.dq, a.dk, a.dv = a.wide[:, :H], a.wide[:, H:2 * H], a.wide[:, 3 * H:]
    a.fwd()
    a.bwd()
    a.check()
    assert all((m[T:] == 7).all() for m in more)


def test_attention_on_two_streams_at_once():
    torch.cuda.synchronize()
    calls = [Attention(attention_inputs(3, 300, 2, 64, torch.float16, "padded", seed=s), p=0.1) for s in range(2)]
    torch.cuda.synchronize()
    for a, stream in zip(calls, [torch.cuda.Stream(), torch.cuda.Stream()]):
        with torch.cuda.stream(stream):
            for _ in range(4):
                a.fwd()
                a.bwd()
    torch.cuda.synchronize()
    for a in calls:
        a.check()


@pytest.mark.parametrize("dt", HALF)
def test_attention_of_the_longest_sequence(dt):
    """65536 tokens, more than 2^32 pairs, with queries, keys and biases of zero: P = 1 / S, each product a mean."""
    S, hd = 65536, 128
    g = torch.Generator().manual_seed(0)
    c = dict(qk=torch.zeros(S, 2 * hd, dtype=dt), qkv=torch.randn(S, 3 * hd, generator=g).to(dt), mask=torch.ones(1, S, dtype=torch.int32),
             table=torch.zeros(64, 1, dtype=dt), buckets=ops.relative_buckets(64, 512), dctx=torch.randn(S, hd, generator=g).to(dt), nh=1, hd=hd, b=1, S=S)
    c["qkv"] += 1
    c["dctx"] += 1
    a = Attention(c)
    a.fwd()
    a.bwd()
    # P and, in the backward pass, P~ are powers of two: exact; fp32 sums of S products of values up to 2^3: 2^-24 S^(1/2) 2^3 of
    # their mean at the most; then one rounding to 16 bits of a value near 1
    tol = u_of(dt) * 1.5 + 2.0 ** -13
    assert (a.ctx.float() - c["qkv"][:, 2 * hd:].double().mean(0).float().to(dev())).abs().max() <= tol
    assert (a.dv.float() - c["dctx"].double().mean(0).float().to(dev())).abs().max() <= tol
    assert not a.dq.any() and not a.dk.any()


def test_attention_same_bits_again():
    c = attention_inputs(3, 200, 2, 64, torch.bfloat16, "holes")
    got = []
    for _ in range(3):
        a = Attention(c, p=0.1)
        a.fwd()
        a.bwd()
        got.append([a.ctx, a.wide, a.dtable])
    for other in got[1:]:
        for x, y in zip(got[0], other):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_attention_of_an_empty_batch():
    e = Attention(attention_inputs(0, 40, 2, 64, torch.bfloat16, poison=False))
    e.fwd()
    e.bwd()
    assert not e.dtable.any()


def test_attention_captured():
    """Forward and backward in a graph, replayed on new inputs; another graph with a workspace of its own beside it."""
    cs = [attention_inputs(2, 90, 2, 64, torch.bfloat16, "padded", seed=s) for s in (1, 2, 3)]
    pair = [Attention(cs[0]), Attention(cs[1])]
    side = torch.cuda.Stream()
    graphs = []
    for a in pair:
        a.fwd()
        a.bwd()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a.fwd()
            a.bwd()
        graphs.append(g)
    for n, t in pair[0].g.items():
        if torch.is_tensor(t):
            t.copy_(cs[2][n])
    pair[0].c = cs[2]
    torch.cuda.synchronize()
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for a in pair:
        a.check()


def _rotary(T, S, nh, hd, dt, with_positions, seed=0):
    g = torch.Generator().manual_seed(seed)
    H = nh * hd
    c = dict(wide=torch.randn(T, 3 * H, generator=g).to(dt), dy=torch.randn(T, 2 * H, generator=g).to(dt),
             gq=(1 + 0.3 * torch.randn(hd, generator=g)).to(dt), gk=(1 + 0.3 * torch.randn(hd, generator=g)).to(dt),
             table=ops.rotary_table(max(S, 64), hd),
             pos=torch.randint(0, 64, (T,), generator=g, dtype=torch.int32) if with_positions else None)
    return c


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,S,nh,hd,pos", [(1, 1, 1, 64, False), (3, 7, 2, 32, False), (2, 5, 3, 128, True), (64, 31, 12, 64, False), (700, 9, 5, 32, True),
                                           (0, 4, 2, 64, False)])
def test_rotary(b, S, nh, hd, pos, dt):
    T, H = b * S, nh * hd
    c = _rotary(T, S, nh, hd, dt, pos)
    d = {n: None if t is None else t.to(dev()) for n, t in c.items()}
    x = d["wide"][:, :2 * H]
    y, wide_dx = torch.empty(T, 2 * H, dtype=dt, device=dev()), torch.full((T, 3 * H), 7.0, dtype=dt, device=dev())
    dgq, dgk = torch.empty_like(d["gq"]), torch.empty_like(d["gk"])
    ws = ops.qk_norm_rotary_workspace(T, nh, hd, dev())
    args = (x, d["gq"], d["gk"], d["table"], S, nh, 1e-6)
    ops.qk_norm_rotary_fwd(*args, y, positions=d["pos"])
    ops.qk_norm_rotary_bwd(d["dy"], *args, ws, wide_dx[:, :2 * H], dgq, dgk, positions=d["pos"])
    at = c["pos"].long() if pos else torch.arange(T) % S
    wy, wdx, wgq, wgk = rotary_64(c["wide"][:, :2 * H], c["gq"], c["gk"], c["table"], at, nh, 1e-6, c["dy"])
    u, f = u_of(dt), 2.0 ** -20
    tiny = torch.finfo(dt).tiny * u
    # fp32 inside (rsqrt 2 ulp, a dozen roundings: 2^-20 of the magnitudes that are added up), one rounding at the end
    heads = lambda t: t.reshape(T, 2, nh, 2, hd // 2)
    mag = heads(wy).square().sum(3, keepdim=True).sqrt().expand(-1, -1, -1, 2, -1).reshape(T, 2 * H)
    assert_within("y", y, wy, u * wy.abs() + f * mag + tiny)
    xh = c["wide"][:, :2 * H].double().reshape(T, 2 * nh, hd)
    r = torch.rsqrt(xh.square().mean(-1, keepdim=True) + 1e-6)
    gain = torch.cat([c["gq"].expand(nh, hd), c["gk"].expand(nh, hd)]).double().abs()
    dyh = c["dy"].double().abs().reshape(T, 2 * nh, 2, hd // 2).sum(2).repeat(1, 1, 2)         # |dn| at most
    size = r * (dyh * gain + (xh * r).abs() * (dyh * gain * (xh * r).abs()).mean(-1, keepdim=True))
    assert_within("dx", wide_dx[:, :2 * H], wdx, u * wdx.abs() + f * size.reshape(T, 2 * H) + tiny)
    part = (dyh * (xh * r).abs()).reshape(T, 2, nh, hd).sum((0, 2))
    for n, got, want, m in (("dgq", dgq, wgq, part[0]), ("dgk", dgk, wgk, part[1])):
        assert_within(n, got, want, u * want.abs() + f * m + tiny)
    assert (wide_dx[:, 2 * H:] == 7.0).all()
    again = d["dy"].clone()
    ops.qk_norm_rotary_bwd(again, *args, ws, again, dgq, dgk, positions=d["pos"])
    assert torch.equal(again, wide_dx[:, :2 * H])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,F", [(1, 8), (7, 512), (33, 200), (300, 1536), (2000, 136), (0, 64)])
def test_gelu8(T, F, dt):
    g = torch.Generator().manual_seed(4)
    x, da = (torch.randn(T, F, generator=g) * 2).to(dt), torch.randn(T, F, generator=g).to(dt)
    bias = torch.randn(F, generator=g).to(dt)
    gx, gda, gb = x.to(dev()), da.to(dev()), bias.to(dev())
    saved, ws = ops.gelu8_saved(T, F, dev()), ops.gelu8_workspace(T, F, dev())
    out, dx, act, db = torch.empty_like(gx), torch.empty_like(gx), torch.empty_like(gx), torch.empty_like(gb)
    ops.gelu8_fwd(gx, gb, out, saved)
    ops.gelu8_bwd(gda, saved, ws, db, dx, act)
    u = u_of(dt)
    tiny = torch.finfo(dt).tiny * u
    want_out = torch.nn.functional.gelu(x.double() + bias.double())
    # x + bias in fp32 (|z| 2^-24, times a slope of up to 1.13); the normal tail within 1.5e-7 / 2 of 1 in 16 bits (erfcf: 2^-22 of itself)
    z = (x.double() + bias.double()).abs()
    tail = 2.0 ** -23 if dt != torch.float32 else 2.0 ** -22
    assert_within("out", out, want_out, u * want_out.abs() + z * (tail + 2.0 ** -23) + tiny)
    # the 8 bits stand for z within half a step, then the backward pass is exact for what they stand for
    held = saved.q.cpu().double() * saved.scale.cpu().double().repeat_interleave(128, 1)[:, :F]
    top = torch.cat([z[:, at:at + 128].amax(1, keepdim=True).expand(-1, min(128, F - at)) for at in range(0, F, 128)], 1) if T else z
    assert_within("held", held, x.double() + bias.double(), top / 254 * (1 + 2.0 ** -20) + z * 2.0 ** -22)
    leaf = held.clone().requires_grad_()
    a = torch.nn.functional.gelu(leaf)
    (wdx,) = torch.autograd.grad(a, leaf, da.double())
    off = 2.0 ** -21 * (1 + held.abs())
    assert_within("act", act, a.detach(), u * a.detach().abs() + off * held.abs().clamp(min=1e-30) + tiny)
    assert_within("dx", dx, wdx, u * wdx.abs() + off * da.double().abs() + tiny)
    wdb = wdx.sum(0)
    assert_within("dbias", db, wdb, u * wdb.abs() + (off * da.double().abs() + 2.0 ** -20 * wdx.abs()).sum(0) + tiny)
    inplace, grad = gx.clone(), gda.clone()
    ops.gelu8_fwd(inplace, gb, inplace, saved)
    ops.gelu8_bwd(grad, saved, ws, db, grad, act)
    assert torch.equal(inplace, out) and torch.equal(grad, dx)


def test_gelu8_edges():
    x = torch.zeros(4, 128, device=dev(), dtype=torch.float32)
    x[1, 5], x[2, 7], x[3, 9] = float("inf"), float("nan"), 1e-35
    saved, ws = ops.gelu8_saved(4, 128, dev()), ops.gelu8_workspace(4, 128, dev())
    out, act, db = torch.empty_like(x), torch.empty_like(x), torch.empty(128, device=dev())
    ops.gelu8_fwd(x, torch.zeros(128, device=dev()), out, saved)
    ops.gelu8_bwd(torch.ones_like(x), saved, ws, db, out, act)
    assert torch.isnan(saved.scale[1:3]).all() and (saved.scale[[0, 3]] == 0).all() and (saved.q == 0).all()
    assert torch.isnan(out[1:3]).all() and (out[[0, 3]] == 0.5).all() and torch.isnan(db).all()


def test_refusals_on_the_device():
    a = Attention(attention_inputs(2, 40, 2, 64, torch.bfloat16))
    small = ops.relative_attention_workspace(1, 40, 2, 64, 9, torch.bfloat16, dev())
    with pytest.raises(ValueError, match="smaller"):
        ops.relative_attention_fwd(a.q, a.k, a.v, *a.args(), a.ctx, small)
    with pytest.raises(ValueError):
        ops.relative_attention_fwd(a.q.float(), a.k.float(), a.v.float(), *a.args(), a.ctx.float(), a.ws)
    with pytest.raises(ValueError):
        ops.relative_attention_fwd(a.q, a.k, a.v, a.g["mask"].cpu(), *a.args()[1:], a.ctx, a.ws)
    with pytest.raises(ValueError):                              # dropout without the seed on the device
        ops.relative_attention_fwd(a.q, a.k, a.v, *a.args()[:4], 0.1, ops.StepRNG(3), 1, a.ctx, a.ws)
    with pytest.raises(ValueError, match="not filled"):          # backward before forward, and behind one of other sizes
        a.bwd()
    a.fwd()
    other = Attention(attention_inputs(1, 40, 2, 64, torch.bfloat16))
    other.ws = a.ws
    with pytest.raises(ValueError, match="not filled"):
        other.bwd()
    n = 65537
    x = torch.zeros(n, 32, dtype=torch.bfloat16, device=dev())
    with pytest.raises(ValueError, match="at most 65536"):
        ops.relative_attention_fwd(x, x.clone(), x.clone(), torch.ones(1, n, dtype=torch.int32, device=dev()), torch.zeros(8, 1, dtype=torch.bfloat16, device=dev()),
                                   a.g["buckets"], 1, 0.0, None, 0, torch.zeros_like(x), a.ws)
    x = torch.zeros(4, 128, device=dev())
    with pytest.raises(ValueError):
        ops.gelu8_fwd(x, torch.zeros(128, device=dev()), x, ops.gelu8_saved(4, 128, "cpu"))
    ops.gelu8_fwd(x, torch.zeros(128, device=dev()), torch.zeros_like(x), saved := ops.gelu8_saved(4, 128, dev()))
    args = (x, saved, ops.gelu8_workspace(4, 128, dev()), torch.zeros(128, device=dev()), torch.zeros_like(x), torch.zeros_like(x))
    ops.gelu8_bwd(*args)
    with pytest.raises(ValueError, match="workspace"):           # the same sizes with a workspace of another type
        ops.gelu8_bwd(*args[:2], args[2].half(), *args[3:])
