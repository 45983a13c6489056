"""The host's part of the training-step operators at its edges, without a GPU: what needs a kernel
is replaced by a stand-in on the CPU."""

from types import SimpleNamespace

import pytest
import torch

CONFIG = SimpleNamespace(hidden_size=16, num_experts=8, num_experts_per_tok=2,
                         moe_intermediate_size=16, norm_topk_prob=True)


class _Experts(torch.nn.Module):
    def forward(self, x, selected, weights):
        assert selected.shape == weights.shape == (x.shape[0], CONFIG.num_experts_per_tok)
        return x * weights.sum(-1, keepdim=True).to(x.dtype)


@pytest.fixture
def layer(monkeypatch):
    """BalancedSparseMoE with a linear router, torch's topk and experts that scale."""
    from spark_gpt_b200 import balanced

    def route(logits, k, **kw):
        return torch.topk(torch.sigmoid(logits.float()), k, -1)
    monkeypatch.setattr(balanced._RouterLogitsFn, "apply", lambda x, w: x @ w.T.to(x.dtype))
    monkeypatch.setattr(balanced, "route_experts", route)
    monkeypatch.setattr(balanced, "_require_cuda", lambda *ts: None)
    moe = balanced.BalancedSparseMoE(CONFIG)
    torch.nn.init.normal_(moe.gate.weight)
    moe.experts = _Experts()
    return moe


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3), (5,), (2, 3)], ids=str)
def test_batches_without_tokens(layer, lead):
    x = torch.randn(*lead, 16)
    out, logits, selected = layer(x)
    assert out.shape == x.shape
    assert logits.shape == (*lead, 8) and selected.shape == (*lead, 2)
    logits, weights, selected = layer.gate(x)
    assert logits.shape == (*lead, 8) and weights.shape == selected.shape == (*lead, 2)
