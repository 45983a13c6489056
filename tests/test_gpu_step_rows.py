"""The training-step operators where a block or a warp goes over several rows, against 64 bits.

The kernels keep to a grid of resident blocks, so with more rows than that holds a group takes
row after row: the places that hold a row, the maxima and lists of its alternatives and what is
read ahead are used again, and column sums run over several rows.  Ordinary rows stand between those
with ties, masks and nothing at all.  Bounds are those of each operator's own tests."""

import math

import pytest
import torch

from oracle import step_oracle as O
from tests import test_gpu_balanced_routing as R
from tests import test_gpu_layer_norm as N
from tests import test_gpu_logprobs as P

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,H", [(40001, 64), (40001, 59), (10007, 1024), (3001, 1001), (1001, 8192),
                                 (1001, 8191), (701, 16384), (701, 12289), (2500, 20001), (5003, 384)])
def test_layer_norm(T, H, dtype):
    N.test_forward_and_gradients(T, H, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", [
    (30001, 256, 8, 8, 4, "top2", "sigmoid", True, True, 2.5),
    (30001, 250, 16, 10, 4, "max", "softmax", True, True, 1.0),
    (40001, 128, 6, 1, 1, "max", "sigmoid", False, True, 1.0),
    (80001, 64, 8, 8, 4, "top2", "softmax", False, False, 1.0),
    (170001, 32, 4, 1, 1, "max", "softmax", True, True, 1.0),
], ids=lambda c: "-".join(map(str, c)))
def test_routing(case, dtype):
    import spark_gpt_b200 as b200
    T, E, k, groups, kept, gs, scoring, bias, normalize, scale = case
    x, b = R.inputs(T, E, dtype, bias, scoring, groups, gs)
    # rows between them: equal logits, a cut set, nothing
    x[5::97] = 0.5
    x[6::97, E // 2:] = -math.inf
    x[7::97] = -math.inf
    kw = dict(bias=b, scoring=scoring, num_groups=groups, kept_groups=kept, group_score=gs,
              normalize=normalize, scale=scale)
    xl = x.clone().requires_grad_(True)
    w, sel = b200.route_experts(xl, k, **kw)
    assert bool(((sel >= 0) & (sel < E)).all())
    assert bool((sel.sort(-1)[0].diff(dim=-1) > 0).all())
    # every row alone gives the same bits, wherever in the grid it was
    at = torch.randperm(T, device=DEV)[:2000]
    w2, sel2 = b200.route_experts(x[at], k, **kw)
    assert torch.equal(sel2, sel[at]) and torch.equal(w2, w[at])
    # the 64-bit choice of ordinary rows, spread over the grid
    plain = torch.ones(T, dtype=torch.bool, device=DEV)
    for r in (5, 6, 7):
        plain[r::97] = False
    some = torch.nonzero(plain)[:, 0][:: 7]
    x64 = x[some].double().requires_grad_(True)
    ref, ref_sel = O.route(x64, k, b, scoring, groups, kept, gs, normalize, scale)
    assert torch.equal(sel[some], ref_sel)
    assert bool(((w[some].double() - ref).abs() <= R.rel(E) * ref.abs()).all())
    dw = torch.randn(T, k, device=DEV)
    w.backward(dw)
    want, = torch.autograd.grad(ref, x64, dw[some].double())
    size = R.grad_scale(O.route_scores(x64.detach(), scoring), sel[some], dw[some], scoring, normalize, scale)
    tol = (2.0 ** -8 if dtype == BF16 else 2 * R.U) * want.abs() + R.rel(E) * size
    assert bool(((xl.grad[some].double() - want).abs() <= tol).all())
    assert not xl.grad[7::97].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,V,top", [(80011, 259, 0), (20011, 259, 5), (40011, 800, 0), (20011, 1500, 32),
                                     (20011, 1500, 0), (15011, 3000, 4), (10007, 12288, 5),
                                     (15011, 4100, 0), (15013, 12300, 3)])
def test_logprobs(T, V, top, dtype):
    x, tok = P.inputs(T, V, dtype, 12)
    x[3::61] = 1.5
    x[4::61] = torch.randint(0, 3, (V,), device=DEV).to(dtype)
    x[5::61, 40:] = -math.inf
    x[6::61, 40:] = torch.finfo(dtype).min
    x[7::61, : V // 2] = -math.inf
    x[8::61] = -math.inf
    x[9::61] = torch.arange(V, device=DEV).to(dtype)
    n = max(1, 40_000_000 // V)
    # the 64-bit form holds a part of the rows at a time; the kernel sees all of them
    whole_forward_and_gradient(x, tok, top, n)


def whole_forward_and_gradient(x, tok, top, n):
    import spark_gpt_b200 as b200
    T, V = x.shape
    gen = torch.Generator(device=DEV).manual_seed(0)
    g = torch.randn(T, device=DEV, generator=gen)
    ge = 0.3 * torch.randn(T, device=DEV, generator=gen)
    xl = x.clone().requires_grad_(True)
    r = b200.token_logprobs(xl, tok, top=top, ignore_index=P.IGNORE)
    d, = torch.autograd.grad((r.logprob, r.entropy), xl, (g, ge))
    for lo in range(0, T, n):
        s = slice(lo, min(T, lo + n))
        xs, ts = x[s], tok[s]
        lp, h, tlp, tids = O.logprobs(xs, ts, top, 1.0, P.IGNORE)
        P.within(r.logprob.detach()[s], lp, P.bound(torch.nan_to_num(lp, 0, 0, 0), V), "logprob")
        P.within(r.entropy.detach()[s], h, 2 * P.bound(h, V) * (1 + h), "entropy")
        if top:
            assert torch.equal(r.top_ids[s], tids)
            P.within(r.top_logprobs[s], tlp, P.bound(torch.nan_to_num(tlp, 0, 0, 0), V), "top")
        want = O.logprob_grads(xs, ts, 1.0, P.IGNORE, g[s], ge[s])
        logp = torch.nan_to_num(torch.log_softmax(xs.double(), -1), 0, 0, -1e4).clamp(-1e4, 0)
        size = logp.exp() * (g[s].abs()[:, None] + ge[s].abs()[:, None] * (logp.abs() + h[:, None].nan_to_num() + 1))
        size = size.scatter_add(1, ts.clamp(0, V - 1)[:, None], g[s].abs()[:, None].double())
        tol = (2.0 ** -8 if x.dtype == BF16 else 2 * P.U) * want.abs().nan_to_num() + 2 * P.bound(logp, V) * size + 2.0 ** -126
        P.within(d[s], want, tol, "d_logits")
