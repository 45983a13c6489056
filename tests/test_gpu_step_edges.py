"""The training-step operators at their edges, on a B200."""

from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def moe(H=256, E=8, k=2, I=128, **kw):
    from spark_gpt_b200 import BalancedSparseMoE
    torch.manual_seed(0)
    m = BalancedSparseMoE(SimpleNamespace(hidden_size=H, num_experts=E, num_experts_per_tok=k,
                                          moe_intermediate_size=I, norm_topk_prob=True, **kw)).to(DEV)
    with torch.no_grad():
        m.gate.weight.normal_(0, 0.05)
        m.experts.gate_up_proj.normal_(0, 0.05)
        m.experts.down_proj.normal_(0, 0.05)
    return m


@pytest.mark.parametrize("shape", [(0, 256), (2, 0, 256), (7, 256), (3, 5, 256)])
def test_balanced_layer_takes_empty_and_ragged_batches(shape):
    """What SparseMoE is held to: shapes kept, zero gradients from no tokens, no fault."""
    from spark_gpt_b200 import _lib
    m = moe()
    x = torch.randn(*shape, device=DEV).to(BF16).requires_grad_(True)
    out, logits, sel = m(x)
    assert out.shape == x.shape
    assert logits.shape == (*shape[:-1], 8) and sel.shape == (*shape[:-1], 2)
    out.float().square().sum().backward()
    before = m.gate.score_bias.clone()
    m.gate.update_bias(sel)
    torch.cuda.synchronize()
    assert _lib.read_fault() == 0
    assert x.grad.shape == x.shape and torch.isfinite(x.grad.float()).all()
    for p in m.parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all()
        if x.numel() == 0:
            assert not p.grad.any()
    if x.numel() == 0:
        assert torch.equal(m.gate.score_bias, before)
