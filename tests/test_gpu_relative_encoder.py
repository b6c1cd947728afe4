"""The three operators of an encoder layer with relative positions as they are used together: the engine's passes on the kernels
against the CPU oracles with the same weights and dropout masks, and training steps eager and from a CUDA graph."""
import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu

from renee_b200 import ops
from renee_b200.models.encoder import EncoderConfig
from renee_b200.models.flat_encoder import FlatEncoder

BASE = EncoderConfig(vocab_size=300, max_position_embeddings=256, dim=128, n_layers=2, n_heads=2, hidden_dim=384, rotary=True,
                     relative_buckets=16, relative_max_distance=40, gelu8=True)


def _passes(cfg, dt, device, ids, mask, d, sd, seed=11):
    enc = FlatEncoder(cfg, device, dt, "mean", seed=3)
    if sd is not None:
        enc.load_encoder_state_dict(sd)
    rng = ops.StepRNG(seed, torch.tensor([seed], dtype=torch.int32, device=device) if device != "cpu" else None)
    e = enc.forward(ids.to(device), mask.to(device), rng, train=True)
    e = e.clone()
    enc.backward(d.to(device).clone())
    return enc, e


@pytest.mark.parametrize("change", [dict(), dict(rotary=False), dict(relative_buckets=0), dict(gelu8=False), dict(dim=256, n_heads=8)])
@pytest.mark.parametrize("b,S", [(6, 20), (3, 200)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_engine_tracks_the_oracles(dt, b, S, change):
    cfg = dataclasses.replace(BASE, **change)
    g = torch.Generator().manual_seed(S)
    mask = (torch.arange(S)[None] < torch.randint(2, S + 1, (b, 1), generator=g)).int()
    ids = torch.randint(1, 300, (b, S), generator=g).int() * mask
    d = torch.randn(b, cfg.dim, generator=g)
    gpu, e_gpu = _passes(cfg, dt, "cuda:0", ids, mask, d, None)
    with torch.no_grad():                                # gains and tables away from their first values, weights exact in 16 bits
        for n in gpu.encoder_param_names:
            t = gpu.view(gpu.p32, n)
            if "_norm" in n or "bias" in n:
                t.add_((torch.randn(t.shape, generator=torch.Generator().manual_seed(len(n))) * 0.3).to(t.device))
        gpu.p32.copy_(gpu.p32.to(dt).float())
    sd = {n: t.cpu() for n, t in gpu.encoder_state_dict().items()}
    gpu, e_gpu = _passes(cfg, dt, "cuda:0", ids, mask, d, sd)
    cpu, e_cpu = _passes(cfg, torch.float32, "cpu", ids, mask, d, sd)
    # about 15 roundings a layer and direction, each within u, on their own: sqrt(2 layers x 2 directions x 15) u in the 2-norm;
    # held pre-activations that a rounding moves to the next step are off by 1/254 of a block's largest, few of them: twice that
    u = torch.finfo(dt).eps / 2
    bound = 2 * 60 ** 0.5 * u
    rel = lambda a, b: ((a.float().cpu() - b).norm() / b.norm()).item()
    assert rel(e_gpu, e_cpu) < bound
    for n in gpu.encoder_param_names:
        want = cpu.view(cpu.g, n)
        if n.endswith("k_lin.bias") and not cfg.rotary and not cfg.relative_buckets:
            continue
        got = gpu.view(gpu.g, n)
        # gradients that cancel (the keys' bias moves all scores of a row alike) are measured beside the layer's other ones
        scale = max(want.norm().item(), 0.05 * cpu.view(cpu.g, n.replace("k_lin", "q_lin")).norm().item())
        assert (got.float().cpu() - want).norm().item() < bound * scale + 1e-6, n


@pytest.mark.parametrize("S", [24, 100])
def test_training_steps_eager_and_captured(S):
    import numpy as np
    from renee_b200.data import xcrepo
    from renee_b200.data.collate import XCCollator
    from renee_b200.data.synthetic import SyntheticSpec, SyntheticXC
    from renee_b200.ops import cuda as cu
    from renee_b200.parallel.dist import DistContext
    from renee_b200.train import TrainConfig, XCTrainer
    from renee_b200.utils.sharding import shard_labels
    L, B = 500, 12
    sh = shard_labels(L, 1)
    spec = SyntheticSpec(num_labels=L, seq_len=S, len_lo=2, len_hi=S, vocab=3000, poisson_lam=2.0, seed=0)
    data = xcrepo.InMemoryDataset(*SyntheticXC(spec).rows(np.arange(6 * B)))
    out = []
    for graph in (False, True):
        cfg = TrainConfig(batch_size=B, epochs=1, seed=0, dropout=0.3, lr1=0.05, lr2=1e-3, warmup=2, wd1=1e-4, noloss=True, fp16xfc=True, maxlen=S,
                          pooling="mean", cuda_graph=graph)
        tr = XCTrainer(cfg, dataclasses.replace(BASE, vocab_size=3000), sh, DistContext(device=torch.device("cuda", 0)), steps_per_epoch=6)
        first = tr.encoder.p32.clone()
        col = XCCollator(sh, data, 0, 1, B, True)
        for k in range(6):
            tr.train_step(col(np.arange(k * B, (k + 1) * B)))
        torch.cuda.synchronize()
        cu.check_status()
        out.append((tr.xfc.W.clone(), tr.encoder.p32.clone()))
        for part in ("q_norm.weight", "relative_bias.weight", "ffn.lin1.weight"):
            n = f"transformer.layer.1.{'attention.' if part[0] in 'qr' else ''}{part}"
            assert not torch.equal(tr.encoder.view(first, n), tr.encoder.view(tr.encoder.p32, n)), f"{n} was not trained"
    # the steps are the same; the embedding gradients are summed by 16-bit atomics in any order
    for a, b in zip(*out):
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 2.0 ** -9


def test_fp32_activations_are_refused():
    with pytest.raises(ValueError, match="16-bit"):
        FlatEncoder(BASE, "cuda:0", torch.float32)
