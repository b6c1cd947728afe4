"""What a workspace of the relative operators is good for: one forward call and its backward calls, whole memory of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from renee_b200 import ops
from tests.relative_cases import attention_inputs
from tests.test_gpu_relative_ops import Attention, dev


def test_a_forward_call_that_failed_leaves_nothing_to_go_back_from(monkeypatch):
    from renee_b200.ops import cuda as cu
    a = Attention(attention_inputs(2, 40, 2, 64, torch.bfloat16))
    a.fwd()
    a.bwd()

    def fails(*args, **kw):
        raise cu.KernelError("refused on the host")

    with monkeypatch.context() as m:
        m.setattr(cu, "_call_typed", fails)
        with pytest.raises(cu.KernelError):
            a.fwd()
    with pytest.raises(ValueError, match="not filled"):
        a.bwd()
    a.fwd()
    a.bwd()
    a.check()


def test_backward_calls_of_another_kind_are_refused():
    a = Attention(attention_inputs(2, 40, 2, 64, torch.bfloat16), p=0.2)
    a.fwd()
    a.bwd()
    for change in (dict(p=0.0), dict(p=0.3), dict(stream=4)):
        was = {n: getattr(a, n) for n in change}
        vars(a).update(change)
        with pytest.raises(ValueError, match="not filled"):
            a.bwd()
        vars(a).update(was)
    a.bwd()
    a.check()
    b = Attention(attention_inputs(2, 40, 2, 64, torch.float16), p=0.2)
    b.ws = a.ws
    with pytest.raises(ValueError, match="not filled"):
        b.bwd()


def test_scratch_and_seeds_without_memory_of_their_own_are_refused(monkeypatch):
    """Scratch whose values share memory counts more of them than there are, an empty seed has none.  (No kernel is launched.)"""
    from renee_b200.ops import cuda as cu
    monkeypatch.setattr(cu, "_call_typed", lambda *a, **k: pytest.fail("a call that should have been refused"))
    x = torch.zeros(8, 256, dtype=torch.bfloat16, device=dev())
    gain, table = torch.zeros(64, dtype=torch.bfloat16, device=dev()), ops.rotary_table(8, 64, device=dev())
    ws = ops.qk_norm_rotary_workspace(8, 2, 64, dev())
    for bad in (ws[:1].expand(ws.numel()), torch.zeros(2 * ws.numel(), device=dev())[::2]):
        with pytest.raises(ValueError, match="workspace"):
            ops.qk_norm_rotary_bwd(x.clone(), x, gain, gain.clone(), table, 8, 2, 1e-6, bad, x.clone(), gain.clone(), gain.clone())
    ws, saved = ops.gelu8_workspace(8, 256, dev()), ops.gelu8_saved(8, 256, dev())
    with pytest.raises(ValueError, match="workspace"):
        ops.gelu8_bwd(x, saved, ws[:1].expand(ws.numel()), torch.zeros(256, dtype=torch.bfloat16, device=dev()), x.clone(), x.clone())
    a = Attention(attention_inputs(2, 40, 2, 64, torch.bfloat16), p=0.2)
    a.rng = ops.StepRNG(5, torch.zeros(0, dtype=torch.int32, device=dev()))
    with pytest.raises(ValueError, match="seed"):
        a.fwd()
