"""Dropout of the relative attention's probabilities where a batch has more of them than there are numbers of 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from renee_b200 import ops
from renee_b200.ops.rng import PairNumbers, mix32
from tests.relative_cases import u_of


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,S,nh", [(1, 65536, 3), (65, 4099, 4)])
def test_no_two_heads_share_their_decisions(b, S, nh, dt):
    """Queries, keys and biases of zero: P = 1 / S, so an output is the mean of the values that were kept, times 2 (p = 0.5)."""
    hd, p, seed, stream, dev = 32, 0.5, 77, 3, torch.device("cuda", 0)
    T, H = b * S, nh * hd
    g = torch.Generator(device=dev).manual_seed(1)
    zero = torch.zeros(T, H, dtype=dt, device=dev)
    v, dctx = ((torch.randn(S, hd, generator=g, device=dev) + 1).to(dt) for _ in range(2))
    wide = lambda t: t.view(1, S, 1, hd).expand(b, S, nh, hd).reshape(T, H)                 # the same for all heads
    rng = ops.StepRNG(seed, torch.tensor([seed], dtype=torch.int32, device=dev))
    args = (zero, zero.clone(), wide(v), torch.ones(b, S, dtype=torch.int32, device=dev), torch.zeros(8, nh, dtype=dt, device=dev),
            ops.relative_buckets(8, 9, dev), nh, p, rng, stream)
    ctx, dq, dk, dv = (torch.empty_like(zero) for _ in range(4))
    dtable = torch.empty(8, nh, dtype=dt, device=dev)
    ws = ops.relative_attention_workspace(b, S, nh, hd, 9, dt, dev)
    ops.relative_attention_fwd(*args, ctx, ws)
    ops.relative_attention_bwd(wide(dctx), *args, ctx, ws, dq, dk, dv, dtable)
    numbers = PairNumbers(stream, S)
    assert numbers.page < b * nh
    # fp32 sums of S products of values up to 2^3: 2^-24 S^(1/2) 2^3 of their mean, P a power of two or (4099) off by u; one rounding at the end
    tol = u_of(dt) * 3 + 2.0 ** -13
    at = torch.arange(S, device=dev)
    for head in sorted({0, 1, nh, numbers.page - 1, numbers.page, b * nh - 1} & set(range(b * nh))):
        number_stream, first = numbers.of(head)
        kept = lambda n: ((mix32(seed, number_stream, n) >> 8).double() / 2 ** 24 >= p).double()
        rows = slice(head // nh * S, (head // nh + 1) * S), slice(head % nh * hd, (head % nh + 1) * hd)
        for i in (0, 1, S // 2 + 1, S - 1):
            want = 2 * (kept(first + i * S + at) @ v.double()) / S
            assert ((ctx[rows][i].double() - want).abs() <= tol * want.abs().clamp(min=1)).all(), (head, i)
            want = 2 * (kept(first + at * S + i) @ dctx.double()) / S
            assert ((dv[rows][i].double() - want).abs() <= tol * want.abs().clamp(min=1)).all(), (head, i)
