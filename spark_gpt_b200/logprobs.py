"""Log probabilities of given tokens, with the entropy and the largest alternatives.

    r = token_logprobs(logits, tokens, top=..., temperature=...)
    r.logprob, r.entropy, r.top_logprobs, r.top_ids

What a loss over given answers needs: -logprob is the cross entropy (the stock model's loss is
train.py:2377-2466), logprob and entropy together a policy gradient's terms; the alternatives
are what a server reports beside a token.  The logits are read once forward and
once backward.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.compiler import is_dynamo_compiling

from . import ops


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                  # (...) fp32
    entropy: torch.Tensor                  # (...) fp32
    top_logprobs: Optional[torch.Tensor]   # (..., top) fp32, None for top = 0
    top_ids: Optional[torch.Tensor]        # (..., top) int64, None for top = 0


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, tokens, top, temperature, ignore):
        logprob, entropy, top_lp, top_ids, stats = ops.token_logprobs_fwd(
            rows, tokens, top, temperature, ignore, True)
        ctx.save_for_backward(rows, tokens, stats, entropy)
        ctx.cfg = (temperature, ignore)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_lp, top_ids)
        return logprob, entropy, top_lp, top_ids

    @staticmethod
    def backward(ctx, d_logprob, d_entropy, _d_top, _d_ids):
        ops.refuse_second_order("token_logprobs")
        if d_logprob is None and d_entropy is None:
            return (None,) * 5
        rows, tokens, stats, entropy = ctx.saved_tensors
        g, ge = (None if d is None else d.float().contiguous() for d in (d_logprob, d_entropy))
        return (ops.token_logprobs_bwd(rows, tokens, stats, entropy, g, ge, *ctx.cfg),) + (
            None,) * 4


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """logits (..., V) bf16 or fp32, tokens (...) int64, over softmax(logits / temperature), the
    temperature from 1e-30 to 1e20.

    Differentiable in the logits through logprob and entropy; the alternatives (the `top` <= 32
    largest logits, equal ones by rising id) are reported only.  A row whose token is
    `ignore_index` is left out: logprob and entropy 0, alternatives (0, -1), no gradient.
    Any other token outside [0, V) gives NaN.  A -inf logit has probability 0 and, unless it is the
    token's, no gradient; a row of -inf alone has log probabilities -inf, entropy 0 and no
    gradient."""
    if is_dynamo_compiling():
        return _outside_graph(logits, tokens, top=top, temperature=temperature,
                              ignore_index=ignore_index)
    rows = ops.as_rows(logits, "token_logprobs")
    lead = logits.shape[:-1]
    if tokens.shape != lead:
        raise ValueError(f"token_logprobs: tokens must have shape {tuple(lead)}, got "
                         f"{tuple(tokens.shape)}")
    if tokens.device != logits.device or tokens.dtype != torch.int64:
        raise RuntimeError("token_logprobs: tokens must be an int64 tensor on the logits' device")
    if not 0 <= top <= min(32, rows.shape[1]):
        raise RuntimeError(f"token_logprobs: need 0 <= top <= min(V, 32), got {top}")
    tokens = tokens.reshape(-1).contiguous()
    args = (rows, tokens, int(top), float(temperature), int(ignore_index))
    if ops.records(rows):
        logprob, entropy, top_lp, top_ids = _TokenLogprobsFn.apply(*args)
    else:
        logprob, entropy, top_lp, top_ids, _ = ops.token_logprobs_fwd(*args, False)
    if len(lead) != 1:
        logprob, entropy = logprob.view(lead), entropy.view(lead)
        if top:
            top_lp, top_ids = top_lp.view(*lead, top), top_ids.view(*lead, top)
    return TokenLogprobs(logprob, entropy, top_lp, top_ids)


_outside_graph = ops.outside_graph(token_logprobs)
