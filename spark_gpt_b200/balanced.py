"""Loss-free balanced routing: sigmoid or softmax scores, a selection bias, expert groups.

    weights, selected = route_experts(logits, top_k, bias=..., ...)   differentiable in logits
    new_bias = balance_bias(bias, selected, rate)
    BalancedSparseMoE(config)          SparseMoE with such a router

Where the stock router (train.py:2134-2158) is softmax -> top-k and balances its experts
through a loss (train.py:3098-3197), here a bias per expert is added to the scores for
the selection alone: after each step it rises by `rate` for experts with fewer
tokens than the mean and falls for those with more.  Experts may come in groups, of which
only the best are searched.
"""

from __future__ import annotations

import torch
import torch.distributed as dist
import torch.nn as nn
from torch.compiler import is_dynamo_compiling

from . import faults, ops
from .moe import Experts, _as_bf16, _extra_logit_grad, _require_cuda

SCORINGS = ("sigmoid", "softmax")
GROUP_SCORES = ("top2", "max")


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, bias, top_k, sigmoid, groups, kept, top2, normalize, scale):
        w, sel = ops.route_experts_fwd(rows, bias, top_k, sigmoid, groups, kept, top2, normalize,
                                       scale)
        ctx.save_for_backward(rows, sel)
        ctx.cfg = (sigmoid, normalize, scale)
        ctx.mark_non_differentiable(sel)
        ctx.set_materialize_grads(False)
        return w, sel

    @staticmethod
    def backward(ctx, d_w, _d_sel):
        ops.refuse_second_order("route_experts")
        if d_w is None:
            return (None,) * 9
        rows, sel = ctx.saved_tensors
        dl = ops.route_experts_bwd(rows, sel, d_w.float().contiguous(), *ctx.cfg)
        return (dl,) + (None,) * 8


def route_experts(logits: torch.Tensor, top_k: int, *, bias: torch.Tensor | None = None,
                  scoring: str = "sigmoid", num_groups: int = 1, kept_groups: int | None = None,
                  group_score: str = "top2", normalize: bool = True, scale: float = 1.0):
    """logits (..., E) bf16 or fp32 -> weights (..., k) fp32, selected (..., k) int64.

    Scores are sigmoid(logits) or softmax(logits), in fp32.  The k experts are the largest
    of score + bias, listed by falling score + bias, equal values by rising index; with
    num_groups > 1 only the experts of the `kept_groups` best groups take part, a group's
    worth being its largest score + bias (group_score "max") or the sum of its two largest
    ("top2").  The weights are the selected scores without the bias, divided by their sum
    (+ 1e-20) with `normalize`, times `scale`.  Differentiable in the logits through the
    weights; the bias has no gradient.  E <= 256, k <= 16, at most 32 groups."""
    if is_dynamo_compiling():
        return _route_outside_graph(logits, top_k, bias=bias, scoring=scoring, num_groups=num_groups,
                                    kept_groups=kept_groups, group_score=group_score,
                                    normalize=normalize, scale=scale)
    if scoring not in SCORINGS:
        raise ValueError(f"route_experts: scoring must be one of {SCORINGS}, got {scoring!r}")
    if group_score not in GROUP_SCORES:
        raise ValueError(f"route_experts: group_score must be one of {GROUP_SCORES}, got "
                         f"{group_score!r}")
    rows = ops.as_rows(logits, "route_experts")
    E = rows.shape[1]
    if not 1 <= top_k <= min(16, E):
        raise RuntimeError(f"route_experts: need 1 <= k <= min(E, 16), got k = {top_k}, E = {E}")
    if bias is not None:
        if bias.shape != (E,):
            raise ValueError(f"route_experts: bias must have shape ({E},), got "
                             f"{tuple(bias.shape)}")
        bias = bias.detach()
        ops._check(bias, torch.float32, "route_experts bias")
        if bias.get_device() != rows.get_device():
            raise RuntimeError(f"route_experts: bias must be on {rows.device}, got {bias.device}")
    args = (top_k, scoring == "sigmoid", num_groups,
            num_groups if kept_groups is None else kept_groups, group_score == "top2",
            bool(normalize), float(scale))
    if ops.records(rows):
        w, sel = _RouteFn.apply(rows, bias, *args)
    else:
        w, sel = ops.route_experts_fwd(rows, bias, *args)
    if logits.dim() == 2:
        return w, sel
    lead = logits.shape[:-1]
    return w.view(*lead, top_k), sel.view(*lead, top_k)


_route_outside_graph = ops.outside_graph(route_experts)


def balance_bias(bias: torch.Tensor, selected: torch.Tensor, rate: float,
                 group=None) -> torch.Tensor:
    """The next selection bias: bias + rate * sign(mean load - load), a new (E,) fp32 tensor.

    A load is the number of times an expert occurs in `selected` (any shape, int64; ids
    outside [0, E) are not counted), summed over the ranks of `group` if one is given."""
    if is_dynamo_compiling():
        return _balance_outside_graph(bias, selected, rate, group)
    if selected.device != bias.device:
        raise RuntimeError(f"balance_bias: selected must be on {bias.device}, got "
                           f"{selected.device}")
    selected = selected.contiguous()
    if group is None:
        return ops.balance_step(bias.detach(), selected, float(rate))
    counts = ops.expert_counts(selected, bias.shape[0])
    dist.all_reduce(counts, group=group)
    return ops.balance_bias(bias.detach(), counts, float(rate))


_balance_outside_graph = ops.outside_graph(balance_bias)


class _RouterLogitsFn(torch.autograd.Function):
    """F.linear of the router (train.py:2145) on the library's GEMMs."""

    @staticmethod
    def forward(ctx, x, w_router):
        _require_cuda(x, w_router)
        faults.raise_pending(x.device)
        E = w_router.shape[0]
        W = ops.router_width(E)
        xb = _as_bf16(x)
        wr = ops.cast_bf16(w_router, W)
        buf = ops.router_logits(xb, wr)
        faults.snapshot(x.device)
        ctx.save_for_backward(xb, wr)
        ctx.cfg = (E, W, x.dtype, w_router.dtype)
        return buf if W == E else buf[:, :E]

    @staticmethod
    def backward(ctx, d_logits):
        xb, wr = ctx.saved_tensors
        E, W, xdtype, wdtype = ctx.cfg
        faults.raise_pending(xb.device)
        if W == E:
            dl = _extra_logit_grad(d_logits, xb.shape[0], W)
        else:  # the products take W columns: zeros beyond E, wherever the gradient's rows lie
            dl = xb.new_zeros(xb.shape[0], W)
            dl[:, :E] = d_logits
        dx = ops.router_dgrad(dl, wr).to(xdtype) if ctx.needs_input_grad[0] else None
        dw = ops.router_wgrad(xb, dl, E).to(wdtype) if ctx.needs_input_grad[1] else None
        faults.snapshot(xb.device)
        return dx, dw


@ops.outside_graph
def _module_outside_graph(module, hidden_states):
    return module.forward(hidden_states)


class BalancedRouter(nn.Module):
    """TopKRouter with ``route_experts``'s selection.

    Beside TopKRouter's fields the config may hold router_scoring ("sigmoid"), n_group (1),
    topk_group (n_group), router_group_score ("top2") and routed_scaling_factor (1.0), with
    those defaults.  ``score_bias`` is a buffer: it is saved with the model and no
    optimizer sees it.  It stays fp32 when the module is cast, since bf16 would lose its steps."""

    def __init__(self, config):
        super().__init__()
        self.num_experts = config.num_experts
        self.top_k = config.num_experts_per_tok
        self.norm_topk_prob = config.norm_topk_prob
        self.scoring = getattr(config, "router_scoring", "sigmoid")
        self.num_groups = getattr(config, "n_group", 1)
        self.kept_groups = getattr(config, "topk_group", self.num_groups)
        self.group_score = getattr(config, "router_group_score", "top2")
        self.scale = getattr(config, "routed_scaling_factor", 1.0)
        self.weight = nn.Parameter(torch.empty(config.num_experts, config.hidden_size))
        self.register_buffer("score_bias", torch.zeros(config.num_experts, dtype=torch.float32))

    def _apply(self, fn, recurse=True):
        bias = self.score_bias
        super()._apply(fn, recurse)
        if self.score_bias.dtype != torch.float32:  # moved, and not cast
            self.score_bias = bias.to(self.score_bias.device)
        return self

    def forward(self, hidden_states: torch.Tensor):
        if is_dynamo_compiling():
            return _module_outside_graph(self, hidden_states)
        shape = hidden_states.shape
        logits = _RouterLogitsFn.apply(hidden_states.reshape(-1, shape[-1]), self.weight)
        w, sel = route_experts(
            logits, self.top_k, bias=self.score_bias, scoring=self.scoring,
            num_groups=self.num_groups, kept_groups=self.kept_groups,
            group_score=self.group_score, normalize=self.norm_topk_prob, scale=self.scale)
        lead = shape[:-1]
        return (logits.view(*lead, logits.shape[-1]), w.view(*lead, self.top_k),
                sel.view(*lead, self.top_k))

    @torch.no_grad()
    def update_bias(self, selected: torch.Tensor, rate: float = 1e-3, group=None) -> None:
        """Move the bias one step toward equal loads, from one step's selections."""
        self.score_bias.copy_(balance_bias(self.score_bias, selected, rate, group))


class BalancedSparseMoE(nn.Module):
    """out, router_logits, selected_experts = BalancedSparseMoE(config)(hidden).

    SparseMoE's call, experts and parameter names with a BalancedRouter; after the step,
    ``moe.gate.update_bias(selected_experts)``."""

    def __init__(self, config):
        super().__init__()
        self.gate = BalancedRouter(config)
        self.experts = Experts(config)

    def forward(self, hidden_states: torch.Tensor):
        if is_dynamo_compiling():
            return _module_outside_graph(self, hidden_states)
        shape = hidden_states.shape
        x = hidden_states.reshape(-1, shape[-1])
        _require_cuda(x)
        logits, w, sel = self.gate(x)
        out = self.experts(x, sel, w)
        lead = shape[:-1]
        return out.view(shape), logits.view(*lead, logits.shape[-1]), sel.view(*lead, sel.shape[-1])
