"""Plain 64-bit forms of the operators of encoder layers with relative positions, and how far 16-bit kernels may be from them."""
import math

import torch

from renee_b200 import ops
from renee_b200.ops.rng import keep_mask

ATTENTION_SHAPES = [  # b, S, nh, hd: one token, tiles of 16, 32, 64 and 128 rows missed and met on both sides, several tiles
    (1, 1, 1, 64), (3, 7, 2, 32), (2, 16, 3, 64), (2, 33, 2, 64), (2, 64, 1, 128), (3, 65, 2, 64), (2, 127, 1, 32), (2, 129, 2, 128),
    (2, 300, 3, 64), (1, 517, 2, 32), (1, 1000, 1, 64)]


def u_of(dt):
    return torch.finfo(dt).eps / 2


def make_mask(kind, b, S, g):
    mask = torch.ones(b, S, dtype=torch.int32)
    if kind in ("padded", "holes", "empty"):
        lens = torch.randint(1, S + 1, (b, 1), generator=g)
        mask = (torch.arange(S)[None] < lens).int()
    if kind == "holes":
        mask *= (torch.rand(b, S, generator=g) > 0.3).int() * 7          # any value but 0 attends
        mask[:, S // 2] = 1
    if kind == "empty":
        mask[b // 2] = 0
    return mask


def attention_inputs(b, S, nh, hd, dt, mask_kind="padded", far=9, buckets=8, seed=0, poison=True):
    """Inputs as views of wider projections, with NaN and infinities in the rows of masked keys."""
    g = torch.Generator().manual_seed(seed)
    T, H = b * S, nh * hd
    mask = make_mask(mask_kind, b, S, g)
    qk, qkv = torch.randn(T, 2 * H, generator=g).to(dt), torch.randn(T, 3 * H, generator=g).to(dt)
    table = (torch.randn(buckets, nh, generator=g)).to(dt)
    dctx = torch.randn(T, H, generator=g).to(dt)
    if poison:
        gone = ((mask == 0) & (mask != 0).any(1, keepdim=True)).view(-1)
        qk[gone, H:] = float("nan")
        qkv[gone, 2 * H:] = float("inf")
    return dict(qk=qk, qkv=qkv, mask=mask, table=table, buckets=ops.relative_buckets(buckets, far), dctx=dctx, nh=nh, hd=hd, b=b, S=S)


def views(c):
    H = c["nh"] * c["hd"]
    return c["qk"][:, :H], c["qk"][:, H:], c["qkv"][:, 2 * H:]


def shut_behind(c, value):
    """Keys behind the query shut out by the table (whose upper half holds their distances); ``value`` None: the type's lowest."""
    half = c["table"].shape[0] // 2
    c["table"][half:] = torch.finfo(c["table"].dtype).min if value is None else value
    return c


def attention_64(c, p=0.0, seed=0, stream=0):
    """Outputs and gradients by autograd in 64 bits, and the bounds of a kernel that holds P and dS in 16 bits (relative error u)
    as operands, ctx in 16 bits inside delta, and everything else in fp32.

    ctx: sum P keep v with P off by u: u sum P keep |v|.  dS = P (dP - delta), delta = dctx ctx with ctx off by u |ctx|: off by
    P u sum |dctx| |ctx|; as an operand by u |dS| more.  dq, dk, dtable: those times |k|, |q|, 1.  fp32: sums of up to a few
    thousand products in chunks, exponentials and logarithms of 2 ulp: f of the sums of magnitudes, f = 2^-14 (scores of up
    to 2^5 in base 2, off by 2^-20 of that)."""
    b, S, nh, hd, dt = c["b"], c["S"], c["nh"], c["hd"], c["qk"].dtype
    u, f = u_of(dt), 2.0 ** -14
    seen = c["mask"] != 0
    some = seen.any(1)
    use = seen | ~some[:, None]
    heads = lambda t: t.double().reshape(b, S, nh, hd).transpose(1, 2)
    q, k, v = (heads(t) for t in views(c))
    k, v = (torch.where(use[:, None, :, None], t, torch.zeros_like(t)) for t in (k, v))
    table = c["table"].double()
    leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
    q, k, v, table = leaves
    far = (c["buckets"].numel() - 1) // 2
    at = torch.arange(S)
    bucket = c["buckets"].long()[(at[None] - at[:, None]).clamp(-far, far) + far]
    s = q @ k.transpose(-1, -2) / math.sqrt(hd) + table[bucket].permute(2, 0, 1)
    s = s.masked_fill(~use[:, None, None, :], -math.inf) * 1.0
    s = torch.where(some[:, None, None, None], s, torch.zeros_like(s))
    w = torch.softmax(s, -1)
    keep = keep_mask(seed, stream, w.shape, p).double() / (1 - p) if p > 0 else torch.ones_like(w)
    ctx = (w * keep) @ v
    do = heads(c["dctx"])
    dq, dk, dv, dtable = torch.autograd.grad(ctx, leaves, do, allow_unused=True)
    out = dict(ctx=ctx.detach(), dq=dq, dk=dk, dv=dv, dtable=dtable)
    q, k, v, w = (t.detach() for t in (q, k, v, w))
    dp = (do @ v.transpose(-1, -2)) * keep
    ds = torch.where(some[:, None, None, None], w * (dp - (dp * w).sum(-1, keepdim=True)), torch.zeros_like(w))
    mag = (do.abs() @ v.abs().transpose(-1, -2)) * keep
    delta = (do.abs() * out["ctx"].abs()).sum(-1, keepdim=True)
    off = torch.where(some[:, None, None, None], u * ds.abs() + w * (u * delta + f * (mag + delta)), torch.zeros_like(w))
    scale = 1 / math.sqrt(hd)
    least = S * torch.finfo(dt).tiny * u * 4 if dt == torch.float16 else 0.0        # fp16: sums of numbers below its normal range
    far_off = dict(ctx=(u + f) * ((w * keep) @ v.abs()), dv=(u + f) * ((w * keep).transpose(-1, -2) @ do.abs()),
                   dq=(off + least) @ k.abs() * scale + f * out["dq"].abs(), dk=(off + least).transpose(-1, -2) @ q.abs() * scale)
    bucket_off = torch.zeros_like(table)
    bucket_off.index_add_(0, bucket.reshape(-1), off.sum(0).permute(1, 2, 0).reshape(S * S, nh))
    rows = lambda t: t.transpose(1, 2).reshape(b * S, nh * hd)
    lim = {n: rows((1 + u) * o + u * out[n].abs() + torch.finfo(dt).tiny * u) for n, o in far_off.items()}
    lim["dtable"] = bucket_off.detach() + u * dtable.abs() + 1e-12
    return {n: (dtable if n == "dtable" else rows(t)) for n, t in out.items()}, lim


def assert_within(name, got, want, limit):
    got = got.detach().double().cpu()
    over = (got - want).abs() - limit
    assert not torch.isnan(got).any(), f"{name} has NaNs"
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{name}: off by {(got - want).abs().flatten()[over.argmax()].item():.3e}, may be {limit.flatten()[over.argmax()].item():.3e}"


def rotary_64(x, gq, gk, table, pos, nh, eps, dy):
    """Output and gradients by autograd in 64 bits, through complex numbers."""
    T, hd = x.shape[0], gq.numel()
    leaves = [t.double().requires_grad_() for t in (x, gq, gk)]
    x, gq, gk = leaves
    turn = torch.complex(*table.double()[pos].chunk(2, -1))[:, None, :]
    parts = []
    for part, gain in zip(x.chunk(2, 1), (gq, gk)):
        t = part.reshape(T, nh, hd)
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * gain
        z = torch.complex(*t.chunk(2, -1)) * turn
        parts.append(torch.cat([z.real, z.imag], -1).reshape(T, nh * hd))
    y = torch.cat(parts, 1)
    return (y.detach(),) + torch.autograd.grad(y, leaves, dy.double())


def gelu8_64(x, bias, da):
    """(gelu(z), held z, its gradient times da, gelu(held z), column sums) in 64 bits; the blocks' scales as fp32 has them."""
    z = x.double() + bias.double()
    T, F = z.shape
    held = torch.empty_like(z)
    for at in range(0, F, 128):
        part = z[:, at:at + 128]
        unit = part.abs().amax(1, keepdim=True) / 127
        held[:, at:at + 128] = torch.where(unit > 0, torch.round(part / unit.clamp(min=1e-300)), torch.zeros_like(part)) * unit
    leaf = held.clone().requires_grad_()
    act = torch.nn.functional.gelu(leaf)
    (dx,) = torch.autograd.grad(act, leaf, da.double())
    return torch.nn.functional.gelu(z), held, dx, act.detach(), dx.sum(0)
