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


def test_balanced_layer_cast_to_bf16():
    """The layer casts its fp32 weights to bf16 itself, so a bf16 module of the same weights gives
    the same bits, and its bias still moves."""
    m, h = moe(), moe()
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(p.to(BF16))
    h.load_state_dict(m.state_dict())
    h.to(BF16)
    x = torch.randn(70, 256, device=DEV).to(BF16)
    dout = torch.randn(70, 256, device=DEV).to(BF16)
    for a, b in zip(m(x), h(x)):
        assert torch.equal(a, b)
    m(x)[0].backward(dout)
    h(x)[0].backward(dout)
    for p, q in zip(m.parameters(), h.parameters()):
        assert q.grad.dtype == BF16
        if p is m.gate.weight:
            assert torch.equal(p.grad.to(BF16), q.grad)
    sel = h(x)[2]
    h.gate.update_bias(sel, rate=1e-3)
    assert h.gate.score_bias.dtype == F32 and float(h.gate.score_bias.abs().max()) == pytest.approx(1e-3)


@pytest.mark.parametrize("E", [60, 64])
def test_log_probabilities_of_the_routers_logits(E):
    """Their gradient's rows lie as the logits' do, W apart: the router's gradients are those of the
    same gradient in contiguous rows."""
    import spark_gpt_b200 as b200
    m = moe(E=E, k=4)
    x = torch.randn(70, 256, device=DEV).to(BF16)
    tokens = torch.randint(E, (70,), device=DEV)

    def grads(contiguous):
        m.zero_grad()
        xl = x.clone().requires_grad_(True)
        logits, _, _ = m.gate(xl)
        r = b200.token_logprobs(logits.contiguous() if contiguous else logits, tokens)
        (r.entropy - r.logprob).sum().backward()
        return xl.grad, m.gate.weight.grad

    for a, b in zip(grads(False), grads(True)):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_gradients_side_by_side_are_clipped_and_shared_ones_refused():
    """Neighbours in one buffer, in any order, share no memory; a tensor that is read twice may be."""
    import spark_gpt_b200 as b200
    big = torch.ones(3000, device=DEV)
    parts = [big[2000:], big[:999], big[999:2000], big[5:5]]
    norm = b200.clip_grads(parts, 1.0)
    assert float(norm) == pytest.approx(3000 ** 0.5)
    assert torch.allclose(big, big.new_tensor(3000 ** -0.5).expand(3000), rtol=1e-6)
    g, out = torch.ones(8, device=DEV), torch.zeros(16, device=DEV)
    assert float(b200.grad_norm([g, g])) == 4.0
    assert float(b200.clip_grads([g, g], 2.0, out=[out[:8], out[8:]])) == 4.0
    assert torch.allclose(out, torch.full_like(out, 0.5), rtol=1e-6) and bool((g == 1).all())
    for grads, o in (([g, g], None), ([g[:5], g[4:]], None), ([g[:4], g[4:]], [g[4:], g[:4]]),
                     ([g, g], [out[:8], out[7:15]])):
        with pytest.raises(RuntimeError, match="overlap"):
            b200.clip_grads(grads, 0.5, out=o)
    assert bool((g == 1).all())
    p = torch.nn.Parameter(torch.zeros(4, device=DEV))
    p.grad = torch.ones(4, device=DEV)
    assert float(b200.clip_grad_norm_([p, p], 1.0)) == 2.0
    assert torch.allclose(p.grad, torch.full_like(p.grad, 0.5), rtol=1e-6)


def test_weight_gradients_of_more_columns_than_half_an_int():
    """2 H passes 31 bits: the weight gradients of one row are products, and found at every column."""
    from spark_gpt_b200 import ops
    H = (1 << 30) + 8
    x = (torch.arange(H, device=DEV, dtype=torch.int32) % 251).to(BF16)[None]
    dy = (torch.arange(H, device=DEV, dtype=torch.int32) % 127).to(BF16)[None]
    stats = torch.tensor([[64.0], [0.5]], device=DEV)
    _, dw, db = ops.layer_norm_bwd(dy, x, None, stats, False, True)
    assert torch.equal(db, dy[0].float())
    assert torch.equal(dw, (x[0].float() - 64.0) * 0.5 * dy[0].float())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("E,k", [(20, 6), (32, 8), (64, 8), (100, 8), (250, 16), (256, 8)])
def test_sigmoid_scores_below_the_smallest_normal_number(E, k, normalize, dtype):
    """Logits from -100 to -84, whose scores pass 2^-126 and are fp32 numbers on the grid of 2^-149: the
    order of the experts, their weights and gradients are those of the definition.  Such a
    score is off by its relative error (rel of test_gpu_balanced_routing.py) and, below 2^-126, by
    3 units of that grid, two of the exponential and one of a product; so are the gradients' terms."""
    import spark_gpt_b200 as b200
    from oracle import step_oracle as O
    from tests.test_gpu_balanced_routing import grad_scale, rel
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.full((9, E), -120.0, device=DEV)
    for t in range(9):
        at = torch.randperm(E, device=DEV, generator=g)[:32]
        x[t, at] = -84.0 - 0.5 * torch.arange(len(at), device=DEV)[torch.randperm(len(at), device=DEV, generator=g)]
    x = x.to(dtype).requires_grad_(True)
    w, sel = b200.route_experts(x, k, normalize=normalize)
    x64 = x.detach().double().requires_grad_(True)
    ref, ref_sel = O.route(x64, k, None, "sigmoid", 1, 1, "max", normalize, 1.0)
    assert torch.equal(sel, ref_sel)
    grid = 3 * 2.0 ** -149 * (1e20 if normalize else 1.0)
    assert bool(((w.double() - ref).abs() <= rel(E) * ref + grid).all()) and bool((w > 0).all())
    dw = torch.randn(9, k, device=DEV, generator=g)
    w.backward(dw)
    want, = torch.autograd.grad(ref, x64, dw.double())
    size = grad_scale(O.route_scores(x64.detach(), "sigmoid"), sel, dw, "sigmoid", normalize, 1.0)
    tol = (2.0 ** -8 if dtype == BF16 else 2.0 ** -23) * want.abs() + rel(E) * size + (
        grid * (1 + dw.abs().amax()) + (2.0 ** -133 if dtype == BF16 else 2.0 ** -149))
    assert bool(((x.grad.double() - want).abs() <= tol).all())
