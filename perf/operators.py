"""Operators of encoder layers with relative positions, as cases that can be timed and compared.

Three operators that one layer of such an encoder uses next to each other, forward and backward:

* ``rotary``  ``ops.qk_norm_rotary_fwd / _bwd``: the queries and keys of every head are divided by their root mean square, scaled
  by a learned vector and rotated by their position;
* ``relative``  ``ops.relative_attention_fwd / _bwd``: attention whose scores carry a learned bias by buckets of the distance
  between key and query, with the gradient of that table;
* ``gelu8``  ``ops.gelu8_fwd / _bwd``: bias + GELU that keeps its pre-activation for the backward pass in 8 bits, and the
  gradient and the recomputed activation from them.

``own`` false computes them from elementary torch operations.  Sizes are those of this repository's encoders (heads of 64 and 32,
widths of the feed-forward blocks), its batches and text lengths, and longer texts.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
BLOCK = 128                                    # values of a row that share a scale in 8 bits
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_PAIRS = {"fwd": 4 * 4099 * 4099 * 12, "step": 32 * 512 * 512 * 16}      # query-key pairs of the largest listed cases
MAX_VALUES = {"rotary": 64 * 509 * 2048, "gelu8": 16384 * 4096}


def _rotary(name, kind, b, S, nh, hd, dtype):
    return dict(name=name, op="rotary", kind=kind, b=b, S=S, nh=nh, hd=hd, dtype=dtype)


def _relative(name, kind, b, S, lo, nh, hd, dtype, p=0.0, holes=False, empty=False):
    return dict(name=name, op="relative", kind=kind, b=b, S=S, lo=lo, nh=nh, hd=hd, dtype=dtype, p=p, buckets=32, far=128,
                holes=holes, empty=empty)


def listed():
    return [
        # one short title through the two-layer encoder: prediction for a single text
        _rotary("rotary_fwd_one_title", "fwd", 1, 7, 2, 64, "bf16"),
        # a training step's batch of titles, both directions
        _rotary("rotary_step_titles", "step", 256, 32, 12, 64, "bf16"),
        # documents whose padded length is no round number, the wider encoder, fp16
        _rotary("rotary_step_documents", "step", 64, 509, 16, 64, "fp16"),
        # one short title again: latency
        _relative("relative_fwd_one_title", "fwd", 1, 7, 7, 2, 64, "bf16"),
        # titles, with dropout of the probabilities as training has it, and a text of which nothing is left
        _relative("relative_step_titles", "step", 256, 32, 6, 12, 64, "bf16", p=0.1, empty=True),
        # abstracts
        _relative("relative_step_s128", "step", 128, 128, 32, 12, 64, "bf16"),
        # full documents on the wider encoder, fp16
        _relative("relative_step_s512", "step", 32, 512, 128, 16, 64, "fp16"),
        # prediction for texts beyond a position table's 512 tokens, odd length
        _relative("relative_fwd_long", "fwd", 4, 4099, 2000, 12, 64, "bf16"),
        # the small encoder's heads of 32, ragged, tokens masked in the middle of texts
        _relative("relative_step_hd32", "step", 45, 301, 40, 12, 32, "bf16", holes=True),
        # one short title through the two-layer encoder's feed-forward block, in the debugging type
        dict(name="gelu8_step_one_title", op="gelu8", kind="step", T=7, F=512, dtype="fp32"),
        # titles through the small encoder's block
        dict(name="gelu8_step_titles", op="gelu8", kind="step", T=8192, F=1536, dtype="bf16"),
        # documents through the wide encoder's block
        dict(name="gelu8_step_documents", op="gelu8", kind="step", T=16384, F=4096, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(("rotary", "relative", "relative", "gelu8"))
    if op == "gelu8":
        F = 8 * _log_int(rng, 8, 512)
        return dict(op=op, kind="step", T=_log_int(rng, 1, MAX_VALUES[op] // F), F=F, dtype=rng.choice(("bf16", "fp16", "fp32")))
    hd = rng.choice((64, 64, 64, 32, 128))
    nh = rng.choice((1, 2, 6, 12, 16))
    kind = rng.choice(("fwd", "step", "step"))
    if op == "rotary":
        S = _log_int(rng, 1, 4096)
        b = _log_int(rng, 1, min(1024, max(1, MAX_VALUES[op] // (S * 2 * nh * hd))))
        return dict(op=op, kind=kind, b=b, S=S, nh=nh, hd=hd, dtype=rng.choice(("bf16", "fp16", "fp32")))
    S = _log_int(rng, 1, 2048 if kind == "step" else 4099)
    b = _log_int(rng, 1, min(512, max(1, MAX_PAIRS[kind] * 64 // (S * S * nh * hd))))
    return dict(op=op, kind=kind, b=b, S=S, lo=rng.randint(1, S), nh=nh, hd=hd, dtype=rng.choice(("bf16", "fp16")),
                p=rng.choice((0.0, 0.0, 0.1)), buckets=rng.choice((32, 32, 16, 64)), far=rng.choice((128, 128, 64, 256)),
                holes=rng.choice((False, False, True)), empty=rng.choice((False, False, True)))


# ------------------------------------------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _bucket_of_distance(buckets, far, device):
    """int32 [2 far + 1]: the bucket of key position - query position = -far .. far.  One half of the buckets for each sign; half
    of those hold one distance each, the others grow with its logarithm up to ``far``."""
    d = torch.arange(-far, far + 1)
    half, exact = buckets // 2, buckets // 4
    n = d.abs().clamp(min=1).double()
    grown = exact + (torch.log(n / exact) / math.log(far / exact) * (half - exact) + 1e-9).floor().long().clamp(max=half - exact - 1)
    return (torch.where(d.abs() < exact, d.abs(), grown) + half * (d > 0)).to(torch.int32).to(device)


def _mask(case, g, dev):
    b, S = case["b"], case["S"]
    lens = torch.randint(case["lo"], S + 1, (b, 1), generator=g, device=dev)
    mask = torch.arange(S, device=dev)[None] < lens
    if case["holes"]:
        mask &= torch.rand(b, S, generator=g, device=dev) > 0.15
    if case["empty"]:
        mask[b // 2] = False
    return mask.to(torch.int32)


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(dtype)

    st = dict(case)
    if case["op"] == "gelu8":
        T, F = case["T"], case["F"]
        # pre-activations of a trained block: mostly a little below zero, a few columns much larger than the others
        spread = torch.exp(0.5 * torch.randn(F, generator=g, device=dev))
        st.update(x=(torch.randn(T, F, generator=g, device=dev) * spread).to(dt), bias=normal(F, mean=-0.4, std=0.3), da=normal(T, F, std=0.05))
        return st
    b, S, nh, hd = (case[k] for k in ("b", "S", "nh", "hd"))
    T, H = b * S, nh * hd
    if case["op"] == "rotary":
        angle = torch.arange(S, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))
        st.update(qkv=normal(T, 3 * H, std=1.2), dy=normal(T, 2 * H, std=0.05), gq=normal(hd, mean=1.0, std=0.2), gk=normal(hd, mean=1.0, std=0.2),
                  table=torch.cat([angle.cos(), angle.sin()], 1).float().to(dev))
        return st
    st.update(qk=normal(T, 2 * H), qkv=normal(T, 3 * H), mask=_mask(case, g, dev), table=normal(case["buckets"], nh, std=0.5),
              bucket=_bucket_of_distance(case["buckets"], case["far"], dev), dctx=normal(T, H, std=0.05),
              seed=torch.randint(1, 2 ** 31 - 1, (1,), generator=g, device=dev, dtype=torch.int32))
    return st


# ------------------------------------------------------------------------------------------------- the framework's calls
class _Seed:
    """The step's dropout seed as the framework's calls take it: on the device."""

    def __init__(self, dev):
        self.dev = dev


def _own_rotary(st):
    from renee_b200 import ops
    T, H, S, nh, hd = st["b"] * st["S"], st["nh"] * st["hd"], st["S"], st["nh"], st["hd"]
    x = st["qkv"][:, :2 * H]
    if "y" not in st:                                  # what a program keeps between steps
        st["y"], st["dx"] = torch.empty_like(st["dy"]), torch.empty_like(st["dy"])
        st["dgq"], st["dgk"] = torch.empty_like(st["gq"]), torch.empty_like(st["gk"])
        st["ws"] = ops.qk_norm_rotary_workspace(T, nh, hd, x.device)
    ops.qk_norm_rotary_fwd(x, st["gq"], st["gk"], st["table"], S, nh, EPS, st["y"])
    if st["kind"] == "fwd":
        return st["y"]
    ops.qk_norm_rotary_bwd(st["dy"], x, st["gq"], st["gk"], st["table"], S, nh, EPS, st["ws"], st["dx"], st["dgq"], st["dgk"])
    return {k: st[k] for k in ("y", "dx", "dgq", "dgk")}


def _own_relative(st):
    from renee_b200 import ops
    b, S, nh, hd = st["b"], st["S"], st["nh"], st["hd"]
    H = nh * hd
    q, k, v = st["qk"][:, :H], st["qk"][:, H:], st["qkv"][:, 2 * H:]
    if "ws" not in st:                                 # what a program keeps between steps
        st["ws"] = ops.relative_attention_workspace(b, S, nh, hd, st["far"], st["qk"].dtype, st["qk"].device)
        st["ctx"], st["dqk"], st["dv"] = torch.empty_like(st["dctx"]), torch.empty_like(st["qk"]), torch.empty_like(st["dctx"])
        st["dtable"], st["rng"] = torch.empty_like(st["table"]), _Seed(st["seed"])
    args = (st["mask"], st["table"], st["bucket"], nh, st["p"], st["rng"], 12)
    ops.relative_attention_fwd(q, k, v, *args, st["ctx"], st["ws"])
    if st["kind"] == "fwd":
        return st["ctx"]
    ops.relative_attention_bwd(st["dctx"], q, k, v, *args, st["ctx"], st["ws"], st["dqk"][:, :H], st["dqk"][:, H:], st["dv"], st["dtable"])
    return {n: st[n] for n in ("ctx", "dqk", "dv", "dtable")}


def _own_gelu8(st):
    from renee_b200 import ops
    x = st["x"]
    if "ws" not in st:                                 # what a program keeps between steps
        st["ws"] = ops.gelu8_workspace(st["T"], st["F"], x.device)
        st["saved"] = ops.gelu8_saved(st["T"], st["F"], x.device)
        st["out"], st["dx"], st["act"] = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        st["dbias"] = torch.empty_like(st["bias"])
    ops.gelu8_fwd(x, st["bias"], st["out"], st["saved"])
    ops.gelu8_bwd(st["da"], st["saved"], st["ws"], st["dbias"], st["dx"], st["act"])
    return {k: st[k] for k in ("out", "dx", "act", "dbias")}


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_rotary(st):
    b, S, nh, hd = st["b"], st["S"], st["nh"], st["hd"]
    T, H, h = b * S, nh * hd, hd // 2
    x = st["qkv"][:, :2 * H].float().view(b, S, 2, nh, hd)
    gain = torch.stack([st["gq"], st["gk"]]).float()[:, None, :]
    cos, sin = st["table"][:, None, None, :h], st["table"][:, None, None, h:]
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    unit = x * r
    n = unit * gain
    y = torch.cat([n[..., :h] * cos - n[..., h:] * sin, n[..., h:] * cos + n[..., :h] * sin], -1).view(T, 2 * H)
    if st["kind"] == "fwd":
        return y.to(st["qkv"].dtype)
    dy = st["dy"].float().view(b, S, 2, nh, hd)
    dn = torch.cat([dy[..., :h] * cos + dy[..., h:] * sin, dy[..., h:] * cos - dy[..., :h] * sin], -1)
    dgain = (dn * unit).sum((0, 1, 3))
    du = dn * gain
    dx = (r * (du - unit * (du * unit).mean(-1, keepdim=True))).view(T, 2 * H)
    dt = st["qkv"].dtype
    return {"y": y.to(dt), "dx": dx.to(dt), "dgq": dgain[0].to(dt), "dgk": dgain[1].to(dt)}


def _kept(seed, stream, n, p):
    """Which of ``n`` numbered elements survive dropout: the step's counter-based rule, in 64-bit integers kept below 2^32."""
    low = 0xFFFFFFFF

    def times(x, c):
        return (x * (c & 0xFFFF) + ((x * (c >> 16) & 0xFFFF) << 16)) & low

    x = (times(torch.arange(n, device=seed.device) & low, 0x9E3779B1) + (seed.long() & low)) & low
    x = times(x ^ (x >> 16), 0x85EBCA6B)
    x = times(x ^ (x >> 13), 0xC2B2AE35)
    x = ((x ^ (x >> 16)) + (stream * 0x27D4EB2F & low)) & low
    x = times(x ^ (x >> 15), 0x2C1B3C6D)
    x = times(x ^ (x >> 12), 0x297A2D39)
    return ((x ^ (x >> 15)) >> 8) >= math.ceil(p * 16777216.0)


def _plain_relative(st):
    b, S, nh, hd, far, p = (st[k] for k in ("b", "S", "nh", "hd", "far", "p"))
    T, H = b * S, nh * hd

    def heads(t):
        return t.float().view(b, S, nh, hd).transpose(1, 2)

    q, k, v = heads(st["qk"][:, :H]), heads(st["qk"][:, H:]), heads(st["qkv"][:, 2 * H:])
    at = torch.arange(S, device=q.device)
    bucket = st["bucket"].long()[(at[None, :] - at[:, None]).clamp(-far, far) + far]                 # [query, key]
    s = q @ k.transpose(-1, -2) / math.sqrt(hd) + st["table"].float()[bucket].permute(2, 0, 1)
    seen = (st["mask"] != 0)[:, None, None, :]
    some = seen.any(-1, keepdim=True)                  # a text of which nothing is left attends to all of its tokens alike
    s = torch.where(some, torch.where(seen, s, torch.full_like(s, -math.inf)), torch.zeros_like(s))
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    keep = _kept(st["seed"], 12, w.numel(), p).view_as(w) / (1.0 - p) if p > 0 else None
    ctx = (w * keep if p > 0 else w) @ v
    dt = st["qk"].dtype

    def rows(t):
        return t.transpose(1, 2).reshape(T, H).to(dt)

    if st["kind"] == "fwd":
        return rows(ctx)
    do = heads(st["dctx"])
    dw = do @ v.transpose(-1, -2)
    if p > 0:
        dw = dw * keep
    dv = (w * keep if p > 0 else w).transpose(-1, -2) @ do
    ds = torch.where(some, w * (dw - (dw * w).sum(-1, keepdim=True)), torch.zeros_like(w))
    dq, dk = ds @ k / math.sqrt(hd), ds.transpose(-1, -2) @ q / math.sqrt(hd)
    dtable = torch.zeros(st["buckets"], nh, device=q.device, dtype=torch.float64)
    dtable.index_add_(0, bucket.view(-1), ds.sum(0, dtype=torch.float64).permute(1, 2, 0).reshape(S * S, nh))
    return {"ctx": rows(ctx), "dqk": torch.cat([rows(dq), rows(dk)], 1), "dv": rows(dv), "dtable": dtable.to(dt)}


def _plain_gelu8(st):
    T, F, dt = st["T"], st["F"], st["x"].dtype
    z = st["x"].float() + st["bias"].float()
    blocks = torch.cat([z, z.new_zeros(T, -F % BLOCK)], 1).view(T, -1, BLOCK)
    top = blocks.abs().amax(-1, keepdim=True)
    q = torch.round(blocks * torch.where(top > 0, 127.0 / top, torch.zeros_like(top)))
    held = (q * (top / 127.0)).view(T, -1)[:, :F]

    def cdf(t):
        return 0.5 * torch.special.erfc(t * -math.sqrt(0.5))

    dx = st["da"].float() * (cdf(held) + held * torch.exp(-0.5 * held * held) / math.sqrt(2.0 * math.pi))
    return {"out": (z * cdf(z)).to(dt), "dx": dx.to(dt), "act": (held * cdf(held)).to(dt), "dbias": dx.sum(0, dtype=torch.float64).to(dt)}


def run(state):
    if own:
        return {"rotary": _own_rotary, "relative": _own_relative, "gelu8": _own_gelu8}[state["op"]](state)
    return {"rotary": _plain_rotary, "relative": _plain_relative, "gelu8": _plain_gelu8}[state["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    step = case["kind"] == "step"
    if case["op"] == "gelu8":
        n = case["T"] * case["F"]
        # forward: x in, activation and 8 bits out; backward: gradient and 8 bits in, gradient and activation out; scales of blocks
        return {"bytes": n * (5 * size + 2 + 8.0 / BLOCK) + 2 * size * case["F"], "flops": 60 * n}
    b, S, nh, hd = (case[k] for k in ("b", "S", "nh", "hd"))
    T, H = b * S, nh * hd
    if case["op"] == "rotary":
        n = 2 * T * H
        return {"bytes": (2 + (3 if step else 0)) * size * n + 4 * S * hd, "flops": (8 + (20 if step else 0)) * n}
    keys = (case["lo"] + S) / 2 * (0.85 if case["holes"] else 1.0)                       # attended ones, expected
    pairs = b * nh * S * keys
    # q, k, v in and ctx out; backward: those and the gradient of ctx in, three gradients out
    return {"bytes": size * T * H * (4 + (8 if step else 0)) + 4 * T, "flops": pairs * hd * (4 + (10 if step else 0))}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rotary(st):
    b, S, nh, hd = st["b"], st["S"], st["nh"], st["hd"]
    H = nh * hd
    x = st["qkv"][:, :2 * H].double().requires_grad_()
    gq, gk = st["gq"].double().requires_grad_(), st["gk"].double().requires_grad_()
    turn = torch.complex(st["table"][:, :hd // 2].double(), st["table"][:, hd // 2:].double()).view(1, S, 1, hd // 2)
    parts = []
    for part, gain in ((x[:, :H], gq), (x[:, H:], gk)):
        t = part.reshape(b, S, nh, hd)
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * gain
        turned = torch.complex(*t.split(hd // 2, -1)) * turn
        parts.append(torch.cat([turned.real, turned.imag], -1).reshape(b * S, H))
    y = torch.cat(parts, 1)
    if st["kind"] == "fwd":
        return y.detach()
    dx, dgq, dgk = torch.autograd.grad(y, (x, gq, gk), st["dy"].double())
    return {"y": y.detach(), "dx": dx, "dgq": dgq, "dgk": dgk}


def _exact_relative(st):
    b, S, nh, hd, far, p = (st[k] for k in ("b", "S", "nh", "hd", "far", "p"))
    H = nh * hd
    qk, v, table = st["qk"].double(), st["qkv"][:, 2 * H:].double(), st["table"].double()
    at = torch.arange(S, device=qk.device)
    bucket = st["bucket"].long()[(at[None, :] - at[:, None]).clamp(-far, far) + far]
    keep = _kept(st["seed"], 12, b * nh * S * S, p).view(b, nh, S, S) if p > 0 else None
    ctx, dqk, dv, dtable = torch.empty_like(v), torch.empty_like(qk), torch.empty_like(v), torch.zeros_like(table)
    for i in range(b):
        attended = st["mask"][i] != 0
        for h in range(nh):
            at_rows, at_q, at_k = slice(i * S, (i + 1) * S), slice(h * hd, (h + 1) * hd), slice(H + h * hd, H + (h + 1) * hd)
            leaves = [t.clone().requires_grad_() for t in (qk[at_rows, at_q], qk[at_rows, at_k], v[at_rows, at_q], table[:, h])]
            q1, k1, v1, t1 = leaves
            if attended.any():
                w = torch.softmax((torch.einsum("id,jd->ij", q1, k1) * hd ** -0.5 + t1[bucket]).masked_fill(~attended, -math.inf), -1)
            else:
                w = torch.full((S, S), 1.0 / S, dtype=torch.float64, device=qk.device)
            o = torch.einsum("ij,jd->id", w if keep is None else w * keep[i, h] / (1.0 - p), v1)
            ctx[at_rows, at_q] = o.detach()
            if st["kind"] == "step":
                got = torch.autograd.grad(o, leaves, st["dctx"][at_rows, at_q].double(), allow_unused=True)
                got = [torch.zeros_like(t) if d is None else d for d, t in zip(got, leaves)]
                dqk[at_rows, at_q], dqk[at_rows, at_k], dv[at_rows, at_q] = got[:3]
                dtable[:, h] += got[3]
    return ctx if st["kind"] == "fwd" else {"ctx": ctx, "dqk": dqk, "dv": dv, "dtable": dtable}


def _exact_gelu8(st):
    x, bias, da = st["x"].double(), st["bias"].double(), st["da"].double()
    T, F = x.shape
    z = x + bias
    held = torch.empty_like(z)
    for at in range(0, F, BLOCK):
        part = z[:, at:at + BLOCK]
        unit = part.abs().amax(1, keepdim=True) / 127.0
        held[:, at:at + BLOCK] = torch.round(part / unit.clamp(min=1e-300)) * unit
    held.requires_grad_()
    act = torch.nn.functional.gelu(held)
    (dx,) = torch.autograd.grad(act, held, da)
    return {"out": torch.nn.functional.gelu(z), "dx": dx, "act": act.detach(), "dbias": dx.sum(0)}


def exact(case, seed):
    if case["op"] == "relative" and case["b"] * case["nh"] > 2048 and case["kind"] == "step" and case["S"] > 64:
        return None                                    # one head at a time: too many of them
    st = prepare(case, seed)
    return {"rotary": _exact_rotary, "relative": _exact_relative, "gelu8": _exact_gelu8}[case["op"]](st)
