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


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(),
                                  lambda m: m.half().bfloat16(), lambda m: m.double()],
                         ids=["to", "bfloat16", "half", "double"])
def test_the_selection_bias_stays_fp32(cast):
    """Its steps of 1e-3 are lost in bf16, and the router takes it in fp32: a cast of the module's
    parameters leaves its type and values."""
    from spark_gpt_b200 import BalancedSparseMoE
    moe = torch.nn.ModuleList([BalancedSparseMoE(CONFIG)])
    gate = moe[0].gate
    gate.score_bias.copy_(1.0 + 0.001 * torch.arange(8))
    want = gate.score_bias.clone()
    cast(moe)
    assert gate.weight.dtype != torch.float32
    assert gate.score_bias.dtype == torch.float32 and torch.equal(gate.score_bias, want)
    assert set(gate.state_dict()) == {"weight", "score_bias"}
    moe.to("meta")
    assert gate.score_bias.device.type == "meta" and gate.score_bias.dtype == torch.float32
    moe.to_empty(device="cpu")
    assert gate.score_bias.device.type == "cpu" and gate.score_bias.dtype == torch.float32


def test_the_selection_bias_is_fp32_whatever_the_default():
    from spark_gpt_b200 import BalancedSparseMoE
    torch.set_default_dtype(torch.bfloat16)
    try:
        moe = BalancedSparseMoE(CONFIG)
    finally:
        torch.set_default_dtype(torch.float32)
    assert moe.gate.score_bias.dtype == torch.float32


@pytest.mark.parametrize("E,W", [(60, 64), (8, 8), (1, 8)])
@pytest.mark.parametrize("stride", ["padded", "contiguous", "wide"])
def test_logit_gradients_reach_the_router_in_its_width(monkeypatch, E, W, stride):
    """A gradient whose rows lie W apart (from a padded copy, or of log probabilities of the router's
    logits) has anything between its rows: the products take W columns, zero beyond E."""
    from spark_gpt_b200 import balanced, faults, ops
    seen = {}
    monkeypatch.setattr(ops, "router_dgrad", lambda dl, wr: seen.setdefault("dgrad", dl) @ wr)
    monkeypatch.setattr(ops, "router_wgrad", lambda x, dl, E: (seen.setdefault("wgrad", dl).T @ x)[:E])
    monkeypatch.setattr(faults, "raise_pending", lambda device: None)
    monkeypatch.setattr(faults, "snapshot", lambda device: None)
    T, H = 6, 16
    xb = torch.randn(T, H).to(torch.bfloat16)
    wr = torch.zeros(W, H, dtype=torch.bfloat16)
    wr[:E] = torch.randn(E, H)
    ld = {"padded": W, "contiguous": E, "wide": W + 8}[stride]
    rows = torch.full((T, ld), float("nan"), dtype=torch.bfloat16)
    rows[:, :E] = torch.randn(T, E)
    d = rows[:, :E]
    ctx = SimpleNamespace(saved_tensors=(xb, wr), cfg=(E, W, torch.bfloat16, torch.float32),
                          needs_input_grad=(True, True))
    dx, dw = balanced._RouterLogitsFn.backward(ctx, d)
    for dl in (seen["dgrad"], seen["wgrad"]):
        assert dl.shape == (T, W) and dl.is_contiguous() and dl.data_ptr() % 16 == 0
        assert torch.equal(dl[:, :E], d) and not dl[:, E:].any()
    assert torch.equal(dx, d.contiguous() @ wr[:E]) and dw.shape == (E, H)
