"""Operators of encoder layers with relative positions, forward and backward.

* :func:`qk_norm_rotary_fwd` / :func:`qk_norm_rotary_bwd`: norms of queries and keys for each head with the rotation by position
  (``csrc/rotary.cu``);
* :func:`relative_attention_fwd` / :func:`relative_attention_bwd`: attention with a learned bias by buckets of the distance between
  key and query, and the gradient of that table (``csrc/relative.cu``);
* :func:`gelu8_fwd` / :func:`gelu8_bwd`: bias + GELU that keeps its pre-activation for the backward pass in 8 bits
  (``csrc/gelu8.cu``).

They write into the caller's buffers like the other ops of the package: kernels for CUDA tensors (on the current stream, without
allocation or synchronisation), the oracles of :mod:`renee_b200.ops.reference` for CPU tensors.  Arguments that neither serves are
refused with a ``ValueError`` on both.  The kernels round to 16 bits what the activations' type is meant for and the products read: P
(unnormalised in the forward pass) and dS; sums, statistics, delta and accumulators are fp32, exponentials good to 2^-22.  The queries'
gradient takes delta from the 16-bit output, the others from the sum it stands for.  A workspace belongs to one call at a time: calls that may overlap on the GPU (two streams,
two captured graphs) take one each.  Results do not depend on the order in which CTAs run: no sum uses atomics.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import reference as ref
from ..utils import guard

HEAD_DIMS = (32, 64, 128)
MAX_DISTANCE = 512                # of the bucket map: the window of sums by distance lives in shared memory
MAX_TOKENS = 65536                # of a sequence on the GPU: its mask lives there too, as bits
MAX_DROPOUT = 0.99                # fp16 probabilities carry 1 / (1 - p) and a power of two up to 2^8 in the backward pass
GELU8_BLOCK = 128                 # neighbouring values of a row that share a scale


_CU = None


def _cuda():
    global _CU
    if _CU is None:
        from . import cuda
        _CU = cuda
    return _CU


def _refuse(cond: bool, what: str) -> None:
    if cond:
        raise ValueError(what)


# Checks that depend on shapes, strides, types, devices and numbers alone are made once for each combination (its key, written out
# in each function: loops over the tensors cost half as much again) and leave the kernels' numbers that follow from it: they cost
# 25 us in Python where the kernels of a small call take 5.  Pointers (alignment, outputs that are inputs) are looked at on every call.
_CHECKED: dict = {}


def _passed(key: tuple, numbers: tuple) -> tuple:
    if len(_CHECKED) >= 4096:
        _CHECKED.clear()
    _CHECKED[key] = numbers
    return numbers


def _sig(*tensors) -> tuple:
    return tuple((t.shape, t.stride(), t.dtype, t.device) for t in tensors)


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _same_place(first: torch.Tensor, **others) -> None:
    for name, t in others.items():
        _refuse(t.device != first.device, f"{name} is on {t.device}, the others on {first.device}")
    if first.is_cuda:
        _refuse(first.device.index != torch.cuda.current_device(),
                f"the tensors are on {first.device}, the current device is cuda:{torch.cuda.current_device()}")


def _rows(name: str, t: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> None:
    """A matrix whose rows may lie apart, in whole 16-byte pieces."""
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols or t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} [{rows}, {cols}], not {t.dtype} {list(t.shape)}")
    size = t.element_size()
    if rows and ((t.stride(1) != 1 and cols > 1) or (rows > 1 and (t.stride(0) * size % 16 or t.stride(0) < cols))):
        raise ValueError(f"{name}: the columns must be adjacent, rows must lie whole 16-byte pieces apart and not overlap")


def _whole(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype) -> None:
    if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} {list(shape)}, not {t.dtype} {list(t.shape)}")


def _pointers(n_out: int, *tensors) -> list:
    """Addresses of the ``n_out`` outputs, then of the inputs.  All must be 16-byte aligned, and no output may start where an input
    or another output does (what one kernel writes a later one would read); tensors without elements have none."""
    at = [t.data_ptr() for t in tensors]
    every = 0
    for a in at:
        every |= a
    _refuse(every & 15 != 0, "every tensor must start on a 16-byte boundary")
    for i in range(n_out):
        if at[i] and at.count(at[i]) > 1:
            raise ValueError("an output is the same memory as another tensor of the call")
    return at


def _head_dim(cols: int, nh: int, on_gpu: bool) -> int:
    _refuse(nh < 1 or cols % nh != 0, f"{cols} columns are no whole number of values for each of {nh} heads")
    hd = cols // nh
    _refuse(hd % 2 != 0 or (on_gpu and hd not in HEAD_DIMS), f"head dim {hd}: the kernels have {HEAD_DIMS}")
    return hd


_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


# ----------------------------------------------------------------------------- q/k norm + rotation
def rotary_table(n_positions: int, hd: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """fp32 ``[n_positions, hd]``: the cosines of a position's ``hd / 2`` angles, then their sines.  Angles in 64 bits: in 32 the
    one of position 100000 is off by 0.004."""
    _refuse(hd % 2 != 0 or n_positions < 1, f"no rotation for head dim {hd} and {n_positions} positions")
    speed = float(base) ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))
    angle = torch.arange(n_positions, dtype=torch.float64)[:, None] * speed
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def _check_rotary(x, gq, gk, table, S, nh, eps, positions, **like_x):
    _refuse(x.dim() != 2 or x.dtype not in _FLOATS or x.shape[1] % (2 * nh if nh > 0 else 1) != 0,
            f"x must be [T, 2 heads head dim] of {[str(d) for d in _FLOATS]}, not {x.dtype} {list(x.shape)}")
    hd = _head_dim(x.shape[1] // 2, nh, x.is_cuda)
    T = x.shape[0]
    for name, t in like_x.items():
        _rows(name, t, T, 2 * nh * hd, x.dtype)
    _rows("x", x, T, 2 * nh * hd, x.dtype)
    _whole("gq", gq, (hd,), x.dtype)
    _whole("gk", gk, (hd,), x.dtype)
    _refuse(table.dim() != 2 or table.shape[0] < 1, "table must have a row for each position")
    _whole("table", table, (table.shape[0], hd), torch.float32)
    _refuse(S < 1 or T % S != 0, f"{T} tokens are no whole number of sequences of {S}")
    if positions is None:
        _refuse(S > table.shape[0], f"table has {table.shape[0]} positions, the sequences {S}")
    else:
        _whole("positions", positions, (T,), torch.int32)
        _same_place(x, positions=positions)
    _refuse(not eps > 0.0, "eps must be above 0")
    _refuse(T * nh * (hd // 16) >= 2 ** 31, f"{T} tokens with {nh} heads of {hd} are too many for one call")
    _same_place(x, gq=gq, gk=gk, table=table, **like_x)
    return hd


def qk_norm_rotary_workspace(T: int, nh: int, hd: int, device) -> torch.Tensor:
    """Scratch of :func:`qk_norm_rotary_bwd` for up to ``T`` tokens (empty on the CPU)."""
    if torch.device(device).type != "cuda":
        return torch.empty(0)
    with torch.cuda.device(device):
        n = _cuda().qk_norm_rotary_blocks(T, nh, hd) * 2 * hd
    return guard.empty(max(n, 1), dtype=torch.float32, device=device, name="qk_norm_rotary.workspace")


def qk_norm_rotary_fwd(x, gq, gk, table, S, nh, eps, out, positions=None) -> None:
    """``x`` ``[T, 2H]`` (queries of all heads, then keys; rows may lie apart) -> ``out``: every head's ``hd`` values divided by
    their root mean square (``eps`` is added to the mean square), times ``gq`` or ``gk`` ``[hd]``, rotated by the token's position:
    value ``i`` with value ``i + hd/2`` by the angle whose cosine and sine ``table`` (:func:`rotary_table`) holds.  Token ``t`` of
    the padded ``[b, S]`` batch stands at ``t % S``, or at ``positions[t]`` (int32; one outside the table counts as its nearest)."""
    key = ("rotary", torch.cuda.current_device() if x.is_cuda else -1, S, nh, eps, x.shape, x.stride(), x.dtype, x.device,
           gq.shape, gq.stride(), gq.dtype, gq.device, gk.shape, gk.stride(), gk.dtype, gk.device, table.shape, table.stride(),
           table.dtype, table.device, out.shape, out.stride(), out.dtype, out.device, None if positions is None else _sig(positions))
    numbers = _CHECKED.get(key)
    if numbers is None:
        hd = _check_rotary(x, gq, gk, table, S, nh, eps, positions, out=out)
        numbers = _passed(key, (_ld(x), _ld(out), (x.shape[0], table.shape[0], S, nh, hd, eps)))
    at = _pointers(1, out, x, gq, gk, table)
    if x.is_cuda:
        return _cuda().qk_norm_rotary_fwd(at, numbers, x, positions)
    out.copy_(ref.qk_norm_rotary_fwd(x, gq, gk, table, S, nh, eps, positions))


def qk_norm_rotary_bwd(dy, x, gq, gk, table, S, nh, eps, ws, dx, dgq, dgk, positions=None) -> None:
    """Gradients of :func:`qk_norm_rotary_fwd` from its own inputs: ``dx`` (may be ``dy`` itself), ``dgq``, ``dgk`` (all written,
    not accumulated)."""
    key = ("rotary'", torch.cuda.current_device() if x.is_cuda else -1, S, nh, eps, x.shape, x.stride(), x.dtype, x.device,
           gq.shape, gq.stride(), gq.dtype, gq.device, gk.shape, gk.stride(), gk.dtype, gk.device, table.shape, table.stride(),
           table.dtype, table.device, dy.shape, dy.stride(), dy.dtype, dy.device, dx.shape, dx.stride(), dx.dtype, dx.device,
           dgq.shape, dgq.stride(), dgq.dtype, dgq.device, dgk.shape, dgk.stride(), dgk.dtype, dgk.device, ws.numel(), ws.is_contiguous(), ws.dtype,
           ws.device, None if positions is None else _sig(positions))
    numbers = _CHECKED.get(key)
    if numbers is None:
        hd = _check_rotary(x, gq, gk, table, S, nh, eps, positions, dy=dy, dx=dx)
        _whole("dgq", dgq, (hd,), x.dtype)
        _whole("dgk", dgk, (hd,), x.dtype)
        _same_place(x, dgq=dgq, dgk=dgk)
        if x.is_cuda:
            need = _cuda().qk_norm_rotary_blocks(x.shape[0], nh, hd) * 2 * hd
            _refuse(ws.numel() < need or not ws.is_contiguous() or ws.device != x.device or ws.dtype != torch.float32,
                    f"the workspace is for fewer tokens: {ws.numel()} values on {ws.device}, the call needs {need} on {x.device}")
        numbers = _passed(key, (_ld(dy), _ld(x), _ld(dx), (x.shape[0], table.shape[0], S, nh, hd, eps)))
    dy_ = dy.data_ptr()
    if dx.data_ptr() == dy_ and dx.stride() == dy.stride():
        at = _pointers(3, dx, dgq, dgk, x, gq, gk, table)
    else:
        at = _pointers(3, dx, dgq, dgk, x, gq, gk, table, dy)
    if x.is_cuda:
        return _cuda().qk_norm_rotary_bwd(at, numbers, dy_, x, ws, positions)
    g = ref.qk_norm_rotary_bwd(dy, x, gq, gk, table, S, nh, eps, positions)
    for out, t in zip((dx, dgq, dgk), g):
        out.copy_(t)


# ----------------------------------------------------------------------------- attention with a bias by buckets of distance
def relative_buckets(num_buckets: int, max_distance: int, device=None) -> torch.Tensor:
    """int32 ``[2 max_distance + 1]``: the bucket of distance (key - query) ``-max_distance .. max_distance``; distances beyond
    count as the ends.  Keys behind the query have the upper half of the buckets; of a half, the first half holds one distance
    each, the others grow with its logarithm and the last one reaches to ``max_distance`` and beyond."""
    half, exact = num_buckets // 2, num_buckets // 4
    _refuse(num_buckets < 4 or num_buckets % 2 != 0 or max_distance <= exact or max_distance > MAX_DISTANCE,
            f"no buckets for {num_buckets} and a distance of {max_distance} (at most {MAX_DISTANCE})")
    out = []
    for d in range(-max_distance, max_distance + 1):
        n = abs(d)
        # the logarithm's steps, with a margin above rounding: at an exact border (n / exact a power of the ratio) the next begins
        grown = exact + int(math.log(n / exact) / math.log(max_distance / exact) * (half - exact) + 1e-9) if n >= exact else n
        out.append(min(grown, half - 1) + (half if d > 0 else 0))
    return torch.tensor(out, dtype=torch.int32, device=device)


class RelativeWorkspace:
    """What :func:`relative_attention_fwd` leaves for its backward pass (``lse``, the biases by distance ``win``, the masks as
    ``bits`` and ``lens``, with the kernels' tile counters behind) and the scratch of that pass (``stats``, ``dwin``)."""

    def __init__(self, lse, win, bits, lens, stats, dwin):
        self.lse, self.win, self.bits, self.lens, self.stats, self.dwin = lse, win, bits, lens, stats, dwin
        self.status = _cuda().workspace(lse.device).status if lse.is_cuda else None      # where waits that run out are noted
        self.sizes = (lse.device, *(t.numel() for t in (lse, win, bits, lens, stats, dwin)))
        self.at = (win.data_ptr(), bits.data_ptr(), lens.data_ptr())
        self.filled = None                                   # what the last forward call was for
        lens.zero_()                                         # before a forward call: nothing that leads out of the buffers


def _relative_sizes(b: int, S: int, nh: int, far: int) -> tuple:
    """Values of the workspace's buffers; the statistics and the bits of a sequence take whole tiles of 128 tokens."""
    cu, up = _cuda(), -(-S // 128) * 128
    return (b * nh * up, nh * cu.relative_window_floats(far, S), b * up // 32, b + 3, 2 * b * nh * (up + 1) + 2,
            b * cu.relative_tiles(S) * nh * (2 * min(far, S - 1) + 1))


def relative_attention_workspace(b: int, S: int, nh: int, hd: int, max_distance: int, dtype, device, scratch=None) -> RelativeWorkspace:
    """Buffers for up to ``b`` sequences of ``S`` tokens.  Each forward call whose backward pass is still to come needs one of its
    own; ``scratch`` (another workspace of the same sizes) lends the buffers that live within one backward call."""
    if torch.device(device).type == "cpu":
        return RelativeWorkspace(*[torch.empty(0)] * 6)
    _refuse(hd not in HEAD_DIMS or dtype not in (torch.bfloat16, torch.float16), f"no kernels for heads of {hd} in {dtype}")
    _refuse(b < 0 or not 1 <= S <= MAX_TOKENS or nh < 1 or not 0 <= max_distance <= MAX_DISTANCE, f"no workspace for {b} x {S} tokens, {nh} heads, distance {max_distance}")
    made = []
    for name, n, dtype in zip(("lse", "win", "bits", "lens", "stats", "dwin"), _relative_sizes(b, S, nh, max_distance),
                              (torch.float32, torch.float32, torch.int32, torch.int32, torch.float32, torch.float32)):
        lent = scratch is not None and name in ("stats", "dwin")
        made.append(getattr(scratch, name) if lent else guard.empty(max(n, 4), dtype=dtype, device=device, name=f"relative_attention.{name}"))
    return RelativeWorkspace(*made)


def _check_relative(q, k, v, mask, table, buckets, nh, p, rng, **like_q):
    _refuse(mask.dim() != 2 or mask.shape[1] < 1, "mask must be [b, S] with S >= 1")
    b, S = mask.shape
    _refuse(q.dim() != 2 or q.dtype not in _FLOATS or (q.is_cuda and q.dtype == torch.float32),
            f"q must be [b S, heads head dim] in 16 bits, not {q.dtype} {list(q.shape)}")
    hd = _head_dim(q.shape[1], nh, q.is_cuda)
    for name, t in dict(q=q, k=k, v=v, **like_q).items():
        _rows(name, t, b * S, nh * hd, q.dtype)
    _whole("mask", mask, (b, S), torch.int32)
    _refuse(table.dim() != 2 or table.shape[0] < 1, "table must be [buckets, heads]")
    _whole("table", table, (table.shape[0], nh), q.dtype)
    n = buckets.numel()
    _refuse(n % 2 == 0 or n > 2 * MAX_DISTANCE + 1, f"buckets must be [2 far + 1] with far <= {MAX_DISTANCE}, not [{n}]")
    _whole("buckets", buckets, (n,), torch.int32)
    _refuse(not 0.0 <= p <= MAX_DROPOUT, f"dropout probability {p}: 0 to {MAX_DROPOUT}")
    _refuse(p > 0.0 and rng is None, "dropout needs the step's seed")
    if q.is_cuda:
        _refuse(p > 0.0 and (rng.dev is None or rng.dev.dtype != torch.int32 or rng.dev.device != q.device or rng.dev.numel() < 1),
                "dropout needs the step's seed as an int32 tensor on the device")
        _refuse(S > MAX_TOKENS, f"sequences of {S} tokens: the kernels have at most {MAX_TOKENS}")
        _refuse(b * nh * ((S + 15) // 16) >= 2 ** 31, f"{b} sequences of {S} tokens with {nh} heads are too many for one call")
    _same_place(q, k=k, v=v, mask=mask, table=table, buckets=buckets, **like_q)
    return b, S, hd


def _seed_sig(p, rng):
    return _sig(rng.dev) if p > 0 and rng is not None and rng.dev is not None else None


def _forward_call(q, sizes, p, stream) -> tuple:
    """What a backward call must have in common with the forward call that filled its workspace.  (That no other call of the same kind
    came between is the caller's to see to, as for the activations themselves.)"""
    return (q.dtype, p, stream if p > 0 else None, *sizes)


def _check_ws(ws, device, need) -> None:
    at, *have = ws.sizes
    _refuse(at != device or any(h < n for h, n in zip(have, need)),
            f"the workspace is for smaller sizes: {have} values on {at}, the call needs {list(need)} on {device}")


def relative_attention_fwd(q, k, v, mask, table, buckets, nh, p, rng, stream, ctx_out, ws) -> None:
    """``ctx = softmax(q k^T / sqrt(hd) + table[buckets[clamp(key - query)], head])`` (dropout of the probabilities) ``v``.

    ``q``, ``k``, ``v`` ``[b S, nh hd]``, biases added, rows may lie apart (views of one projection); ``mask`` ``[b, S]`` int32, 0 =
    masked key: it counts as absent, whatever its row holds.  A sequence without any attended key attends to all of its tokens
    alike, as :func:`renee_b200.ops.attention_fwd` has it.  A distance whose table entry is minus infinity (or beyond -2.3e38) is
    not attended at; a query to which nothing else is left gives NaN.  ``table`` ``[buckets, nh]`` in the activations' type, ``buckets`` from
    :func:`relative_buckets` (or any int32 map of ``2 far + 1`` distances).  Dropout decisions are those of
    :class:`renee_b200.ops.rng.PairNumbers`.  ``ctx_out`` ``[b S, nh hd]``, contiguous.  ``ws``
    (:func:`relative_attention_workspace`) receives what the backward pass needs."""
    key = ("relative", torch.cuda.current_device() if q.is_cuda else -1, nh, p, q.shape, q.stride(), q.dtype, q.device,
           k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, mask.shape, mask.stride(), mask.dtype,
           mask.device, table.shape, table.stride(), table.dtype, table.device, buckets.shape, buckets.stride(), buckets.dtype,
           buckets.device, ctx_out.shape, ctx_out.stride(), ctx_out.dtype, ctx_out.device, ws.sizes, _seed_sig(p, rng))
    numbers = _CHECKED.get(key)
    if numbers is None:
        b, S, hd = _check_relative(q, k, v, mask, table, buckets, nh, p, rng)
        _whole("ctx_out", ctx_out, (b * S, nh * hd), q.dtype)
        _same_place(q, ctx_out=ctx_out)
        far = (buckets.numel() - 1) // 2
        if q.is_cuda:
            _check_ws(ws, q.device, _relative_sizes(b, S, nh, far)[:4])
        numbers = _passed(key, (_ld(q), _ld(k), _ld(v), (far, table.shape[0], b, S, nh, hd)))
    at = _pointers(1, ctx_out, q, k, v, table)
    if q.is_cuda:
        ws.filled = None                                     # a call that fails leaves nothing to go back from
        _cuda().relative_attention_fwd(at, numbers, q, mask, buckets, p, rng, stream, ws)
        ws.filled = _forward_call(q, numbers[3], p, stream)
        return
    ctx_out.copy_(ref.relative_attention_fwd(q, k, v, mask, table, buckets, nh, p, rng.seed if p > 0 else 0, stream))


def relative_attention_bwd(dctx, q, k, v, mask, table, buckets, nh, p, rng, stream, ctx, ws, dq, dk, dv, dtable) -> None:
    """Gradients of :func:`relative_attention_fwd` from its inputs, its output ``ctx`` and the workspace it filled: ``dq``, ``dk``,
    ``dv`` (rows may lie apart) and ``dtable`` ``[buckets, nh]``, all written, not accumulated.  May be called again.  The last forward
    call on ``ws`` must have been the one with these inputs: one of other sizes, another type, dropout or stream of decisions, or one
    that failed is refused, but another call of the same kind (an evaluation between the passes) cannot be told from it."""
    key = ("relative'", torch.cuda.current_device() if q.is_cuda else -1, nh, p, q.shape, q.stride(), q.dtype, q.device,
           k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, mask.shape, mask.stride(), mask.dtype,
           mask.device, table.shape, table.stride(), table.dtype, table.device, buckets.shape, buckets.stride(), buckets.dtype,
           buckets.device, dctx.shape, dctx.stride(), dctx.dtype, dctx.device, ctx.shape, ctx.stride(), ctx.dtype, ctx.device,
           dq.shape, dq.stride(), dq.dtype, dq.device, dk.shape, dk.stride(), dk.dtype, dk.device, dv.shape, dv.stride(), dv.dtype,
           dv.device, dtable.shape, dtable.stride(), dtable.dtype, dtable.device, ws.sizes, _seed_sig(p, rng))
    numbers = _CHECKED.get(key)
    if numbers is None:
        b, S, hd = _check_relative(q, k, v, mask, table, buckets, nh, p, rng, dq=dq, dk=dk, dv=dv)
        _whole("dctx", dctx, (b * S, nh * hd), q.dtype)
        _whole("ctx", ctx, (b * S, nh * hd), q.dtype)
        _whole("dtable", dtable, tuple(table.shape), q.dtype)
        _same_place(q, dctx=dctx, ctx=ctx, dtable=dtable)
        far = (buckets.numel() - 1) // 2
        if q.is_cuda:
            _check_ws(ws, q.device, _relative_sizes(b, S, nh, far))
        numbers = _passed(key, (_ld(q), _ld(k), _ld(v), (far, table.shape[0], b, S, nh, hd), _ld(dq), _ld(dk), _ld(dv)))
    at = _pointers(4, dq, dk, dv, dtable, q, k, v, dctx, ctx, table)
    if q.is_cuda:
        _refuse(ws.filled != _forward_call(q, numbers[3], p, stream),
                "the workspace was not filled by a forward call of these sizes, type, dropout and stream of decisions")
        return _cuda().relative_attention_bwd(at, numbers, q, buckets, p, rng, stream, ws)
    g = ref.relative_attention_bwd(dctx, q, k, v, mask, table, buckets, nh, p, rng.seed if p > 0 else 0, stream)
    for out, t in zip((dq, dk, dv, dtable), g):
        out.copy_(t)


# ----------------------------------------------------------------------------- bias + GELU with its pre-activation in 8 bits
@dataclass
class Gelu8Saved:
    """A pre-activation in 8 bits: ``q`` int8 ``[T, F]`` and ``scale`` fp32 ``[T, ceil(F / 128)]``; it stands for ``q scale``."""
    q: torch.Tensor
    scale: torch.Tensor

    def __getitem__(self, rows) -> "Gelu8Saved":
        return Gelu8Saved(self.q[rows], self.scale[rows])


def gelu8_saved(T: int, F: int, device) -> Gelu8Saved:
    return Gelu8Saved(guard.empty(T, F, dtype=torch.int8, device=device, name="gelu8.saved"),
                      guard.empty(T, -(-F // GELU8_BLOCK), dtype=torch.float32, device=device, name="gelu8.scale"))


def gelu8_workspace(T: int, F: int, device) -> torch.Tensor:
    """Scratch of :func:`gelu8_bwd` for up to ``T`` rows (empty on the CPU)."""
    if torch.device(device).type != "cuda":
        return torch.empty(0)
    with torch.cuda.device(device):
        n = _cuda().gelu8_splits(T, F) * F
    return guard.empty(max(n, 1), dtype=torch.float32, device=device, name="gelu8.workspace")


def _check_gelu8(saved, **like_x):
    x = next(iter(like_x.values()))
    _refuse(x.dim() != 2 or x.dtype not in _FLOATS or x.shape[1] % 8 != 0 or x.shape[1] < 8,
            f"rows must be a multiple of 8 values of {[str(d) for d in _FLOATS]}, not {x.dtype} {list(x.shape)}")
    T, F = x.shape
    for name, t in like_x.items():
        _whole(name, t, (T, F), x.dtype)
    _whole("saved.q", saved.q, (T, F), torch.int8)
    _whole("saved.scale", saved.scale, (T, -(-F // GELU8_BLOCK)), torch.float32)
    _refuse(T >= 2 ** 30 or F >= 2 ** 30, f"{T} rows of {F} are too many for one call")
    _same_place(x, **{"saved.q": saved.q, "saved.scale": saved.scale}, **like_x)
    return T, F


def gelu8_fwd(x, bias, out, saved) -> None:
    """``out = gelu(x + bias)`` for ``x`` ``[T, F]`` (erf GELU); ``saved`` receives ``x + bias`` in 8 bits: 128 neighbouring
    values of a row share a scale and are held to 1/254 of the largest of them.  The normal tail is good to 1.5e-7 of 1 for 16-bit
    outputs, as in :func:`renee_b200.ops.bias_gelu_fwd` (so fp16 ones below z = -3.5 are off by more than their rounding).  A block with an infinity or a NaN stands
    for NaNs.  ``out`` may be ``x`` itself."""
    q, scale = saved.q, saved.scale
    key = ("gelu8", torch.cuda.current_device() if x.is_cuda else -1, x.shape, x.stride(), x.dtype, x.device, bias.shape, bias.stride(),
           bias.dtype, bias.device, out.shape, out.stride(), out.dtype, out.device, q.shape, q.stride(), q.dtype, q.device, scale.shape,
           scale.stride(), scale.dtype, scale.device)
    if key not in _CHECKED:
        T, F = _check_gelu8(saved, x=x, out=out)
        _whole("bias", bias, (F,), x.dtype)
        _same_place(x, bias=bias)
        _passed(key, ())
    x_, q_ = x.data_ptr(), q.data_ptr()
    at = _pointers(1, out, bias) if out.data_ptr() == x_ else _pointers(1, out, bias, x)
    _refuse(q_ % 8 != 0, "saved.q must start on an 8-byte boundary")
    if x.is_cuda:
        return _cuda().gelu8_fwd(x, x_, at[1], at[0], q_, scale)
    y, q8, s8 = ref.gelu8_fwd(x, bias)
    out.copy_(y); q.copy_(q8); scale.copy_(s8)


def gelu8_bwd(da, saved, ws, dbias, dx, act_out) -> None:
    """From the gradient ``da`` of the activation and the 8 bits: ``dx = da gelu'(z)``, its column sums ``dbias``, and the
    activation ``act_out = gelu(z)`` again (for the weight gradient of the linear that read it).  ``dx`` may be ``da`` itself."""
    q, scale = saved.q, saved.scale
    key = ("gelu8'", torch.cuda.current_device() if da.is_cuda else -1, da.shape, da.stride(), da.dtype, da.device, q.shape, q.stride(),
           q.dtype, q.device, scale.shape, scale.stride(), scale.dtype, scale.device, dbias.shape, dbias.stride(), dbias.dtype,
           dbias.device, dx.shape, dx.stride(), dx.dtype, dx.device, act_out.shape, act_out.stride(), act_out.dtype, act_out.device,
           ws.numel(), ws.is_contiguous(), ws.dtype, ws.device)
    if key not in _CHECKED:
        T, F = _check_gelu8(saved, da=da, dx=dx, act_out=act_out)
        _whole("dbias", dbias, (F,), da.dtype)
        _same_place(da, dbias=dbias)
        if da.is_cuda:
            need = _cuda().gelu8_splits(T, F) * F
            _refuse(ws.numel() < need or not ws.is_contiguous() or ws.device != da.device or ws.dtype != torch.float32,
                    f"the workspace is for fewer rows: {ws.numel()} values on {ws.device}, the call needs {need} on {da.device}")
        _passed(key, ())
    da_, dx_, q_ = da.data_ptr(), dx.data_ptr(), q.data_ptr()
    at = _pointers(2, act_out, dbias, da) if dx_ == da_ else _pointers(3, act_out, dbias, dx, da)
    _refuse(q_ % 8 != 0, "saved.q must start on an 8-byte boundary")
    if da.is_cuda:
        return _cuda().gelu8_bwd(da, da_, q_, scale, ws, at[1], dx_, at[0])
    d, a, db = ref.gelu8_bwd(da, q, scale)
    dx.copy_(d); act_out.copy_(a); dbias.copy_(db)
