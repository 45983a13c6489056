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


@pytest.fixture
def plain_operators(monkeypatch):
    """The launches replaced by plain forward formulas, so that the calls run on the CPU."""
    from spark_gpt_b200 import ops
    monkeypatch.setattr(ops, "as_rows", lambda t, name: t)
    monkeypatch.setattr(ops, "aligned_rows", lambda t: t)
    monkeypatch.setattr(ops, "layer_norm_fwd", lambda x, w, b, eps, save, like=None: (
        torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, eps), x.new_zeros(2, x.shape[0])))
    monkeypatch.setattr(ops, "route_experts_fwd", lambda x, bias, k, *cfg: torch.topk(torch.sigmoid(x), k))
    monkeypatch.setattr(ops, "token_logprobs_fwd", lambda x, tokens, *cfg: (
        x.log_softmax(-1).gather(1, tokens[:, None])[:, 0], x.sum(-1), None, None, x.new_zeros(x.shape[0], 2)))


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", ["norm", "norm weight", "norm bias", "route", "logprob"])
def test_forward_mode_is_refused(plain_operators, which, grad_mode):
    """The operators have no forward-mode derivative: a tangent is an error, as it is in the
    layer, and is not dropped (which would read as zero)."""
    import torch.autograd.forward_ad as fwd

    import spark_gpt_b200 as b200
    x, w, b = torch.randn(4, 8), torch.randn(8), torch.randn(8)
    tokens = torch.zeros(4, dtype=torch.int64)
    calls = {"norm": lambda f: b200.layer_norm(f(x), w, b), "norm weight": lambda f: b200.layer_norm(x, f(w), b),
             "norm bias": lambda f: b200.layer_norm(x, w, f(b)), "route": lambda f: b200.route_experts(f(x), 2),
             "logprob": lambda f: b200.token_logprobs(f(x), tokens)}
    with torch.set_grad_enabled(grad_mode):
        calls[which](lambda t: t)
        with fwd.dual_level():
            calls[which](lambda t: t)  # without a tangent nothing changes
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                calls[which](lambda t: fwd.make_dual(t, torch.ones_like(t)))


def test_gradient_lists_refuse_tangents(monkeypatch):
    import torch.autograd.forward_ad as fwd

    from spark_gpt_b200 import ops
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    g = torch.randn(4)
    with fwd.dual_level():
        ops.GradList([g], "grad_norm")
        with pytest.raises(RuntimeError, match="grad_norm: .*forward-mode"):
            ops.GradList([g, fwd.make_dual(g, torch.ones(4))], "grad_norm")


@pytest.fixture(scope="module")
def call():
    from spark_gpt_b200 import _lib
    from spark_gpt_b200.build import build
    build()
    return _lib.call


MiB = 1 << 20


@pytest.mark.parametrize("entry", ["b200moe_grad_clip", "b200moe_clip_grads"])
@pytest.mark.parametrize("grads,out,sizes,kinds", [
    ([MiB, MiB], None, [8, 8], [1, 1]),                           # the same tensor twice
    ([MiB, 2 * MiB, 3 * MiB, MiB], None, [8, 8, 8, 4], [1] * 4),  # again, with others between
    ([MiB, MiB + 12], None, [4, 8], [1, 1]),                      # an end in the next one's start
    ([2 * MiB, MiB], None, [4, MiB // 4 + 1], [1, 1]),            # the same in falling order
    ([MiB, MiB + 64, MiB + 128], None, [1000, 2, 2], [0, 0, 0]),  # two inside a first
    ([MiB, 2 * MiB], [3 * MiB, 3 * MiB + 8], [8, 8], [0, 0]),     # outputs into each other
    ([MiB, 2 * MiB], [3 * MiB, MiB], [8, 8], [1, 1]),             # an output into another gradient
    ([MiB], [MiB + 4], [8], [1]),                                 # into its own, shifted
    ([MiB, MiB], [MiB, 2 * MiB], [8, 8], [1, 1]),                 # one read, the same written
], ids=str)
def test_gradients_that_share_memory_are_refused(call, entry, grads, out, sizes, kinds):
    """Blocks that scale them would write the same elements.  Nothing is launched."""
    from array import array
    g, o, n, f = array("q", grads), array("q", out or grads), array("q", sizes), array("i", kinds)
    at = lambda a: a.buffer_info()[0]  # noqa: E731
    tail = (16, 592, 1.0, 16, None) if entry == "b200moe_grad_clip" else (16, 1.0, 16, None)
    with pytest.raises(RuntimeError, match="overlap"):
        call(entry, at(g), at(o), at(n), at(f), len(grads), 0, *tail)


def test_a_parameter_listed_twice_counts_once(monkeypatch):
    """Tied weights reach a list of parameters by two names; the gradient is one."""
    import spark_gpt_b200 as b200
    from spark_gpt_b200 import ops
    seen = []
    monkeypatch.setattr(ops, "GradList", lambda tensors, name: SimpleNamespace(tensors=tensors))
    monkeypatch.setattr(ops, "clip_grads", lambda g, out, inf, m: seen.append(g.tensors))
    a, b, c = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    for p in (a, b, c):
        p.grad = torch.ones(3)
    b200.clip_grad_norm_([a, b, a, c, b], 1.0)
    b200.clip_grad_norm_([a, b, a], 1.0, sharded=[c, a, c])
    assert [[id(t) for t in s] for s in seen] == [[id(p.grad) for p in (a, b, c)], [id(p.grad) for p in (b, c, a)]]


@pytest.mark.parametrize("temperature", [1e21, 1e30, 3e38, float("inf"), 1e-31, 1e-38, 1e-42, 0.0, -1.0,
                                         float("nan")])
def test_temperatures_beyond_the_arithmetic_are_refused(call, temperature):
    """From 1e-30 to 1e20 the scales and their products with the floor of the logits are fp32 numbers;
    beyond, a padding place or a -inf logit would have probability."""
    with pytest.raises(RuntimeError, match="temperature"):
        call("b200moe_token_logprobs_fwd", 16, 0, 100, 16, 4, 100, temperature, -100, 0, 16, 16, None, None,
             None, None)
    with pytest.raises(RuntimeError, match="temperature"):
        call("b200moe_token_logprobs_bwd", 16, 0, 100, 16, 4, 100, temperature, -100, 16, 16, 16, 16, 16, 100,
             None)


@pytest.mark.parametrize("columns", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 8])
def test_more_columns_than_an_int_holds_are_refused(call, columns):
    """The entry points take the columns as 32 bits, in which 2^32 + 8 would be 8."""
    from spark_gpt_b200 import ops
    rows = SimpleNamespace(is_cuda=True, dtype=torch.bfloat16, shape=(1, columns), dim=lambda: 2,
                           stride=lambda d: (columns, 1)[d])
    if columns < 2 ** 31:
        assert ops.as_rows(rows, "norm") is rows
        with pytest.raises(RuntimeError, match="H <="):
            call("b200moe_layer_norm_fwd", 16, 0, columns, None, None, 1, columns, 1e-5, 16, None, None, None)
        with pytest.raises(RuntimeError, match="H <="):
            call("b200moe_layer_norm_bwd", 16, columns, 16, 0, columns, None, 16, 16, 1, columns, 16, None,
                 None, None, 0, None)
    else:
        with pytest.raises(RuntimeError, match="norm: .*columns"):
            ops.as_rows(rows, "norm")


def test_statistics_off_their_alignment_are_refused(call):
    """The log probabilities' statistics are read and written as pairs of fp32."""
    with pytest.raises(RuntimeError, match="stats"):
        call("b200moe_token_logprobs_fwd", 16, 0, 100, 16, 4, 100, 1.0, -100, 0, 16, 16, None, None, 20, None)
    with pytest.raises(RuntimeError, match="stats"):
        call("b200moe_token_logprobs_bwd", 16, 0, 100, 16, 4, 100, 1.0, -100, 20, 16, 16, 16, 16, 100, None)


@pytest.mark.parametrize("how", ["clip_grads", "out", "clip_grad_norm_"])
def test_autograd_sees_that_gradients_were_scaled(monkeypatch, how):
    """What is scaled in place may be held by a graph (of a penalty on the gradients): its backward is an
    error then, as after any in-place operation, and is not that of the scaled values."""
    import spark_gpt_b200 as b200
    from spark_gpt_b200 import ops
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(ops, "_call_on", lambda *args: None)
    monkeypatch.setattr(ops, "_grad_partials_count", lambda: 592)
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad, other = torch.ones(4), torch.ones(4)
    penalty = (torch.ones(4, requires_grad=True) * p.grad).sum()
    result = (torch.ones(4, requires_grad=True) * other).sum()
    if how == "clip_grads":
        b200.clip_grads([p.grad], 0.5)
    elif how == "out":
        b200.clip_grads([p.grad], 0.5, out=[other])
    else:
        b200.clip_grad_norm_([p], 0.5)
    changed, kept = (result, penalty) if how == "out" else (penalty, result)
    kept.backward()
    with pytest.raises(RuntimeError, match="inplace operation"):
        changed.backward()
