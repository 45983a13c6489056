"""The global gradient norm over many tensors, and clipping.

    norm = clip_grad_norm_(model.parameters(), 1.0)     before optimizer.step()
    norm = clip_grads(grads, 1.0, out=buffers)          gradients in hand, in place or not
    norm = grad_norm(grads)

Nothing waits for the GPU: the norm stays on the device, and the scaling reads it there.
"""

from __future__ import annotations

import math

import torch
import torch.distributed as dist

from . import ops


def _inf(norm_type) -> bool:
    if norm_type not in (2, 2.0, math.inf):
        raise ValueError(f"gradient norm: norm_type must be 2 or inf, got {norm_type!r}")
    return norm_type == math.inf


@ops.outside_graph
@torch.no_grad()
def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """sqrt of the sum of squares (or, for norm_type inf, the largest magnitude) of all
    tensors' elements: a 0-d fp32 tensor.  bf16 or fp32 contiguous CUDA tensors."""
    inf_norm = _inf(norm_type)
    grads = ops.GradList(list(grads), "grad_norm")
    if not grads.tensors:
        raise ValueError("grad_norm: no tensors")
    return ops.grad_clip(None, inf_norm, ops.grad_partials(grads, inf_norm), 0.0)


@ops.outside_graph
@torch.no_grad()
def clip_grads(grads, max_norm: float, *, out=None, norm_type: float = 2.0) -> torch.Tensor:
    """Scale the gradients by min(1, max_norm / (norm + 1e-6)), in place or into the tensors
    `out` (same sizes and types); returns the norm before clipping (0-d fp32).  What is written
    shares no memory with another tensor of either list.

    Where the norm is not finite the gradients keep their values: the caller decides on the
    returned norm whether to take the step."""
    inf_norm = _inf(norm_type)
    grads = ops.GradList(list(grads), "clip_grads")
    if not grads.tensors:
        raise ValueError("clip_grads: no tensors")
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grads: max_norm must not be negative, got {max_norm!r}")
    dst = grads
    if out is not None:
        dst = ops.GradList(list(out), "clip_grads out")
        if (dst.sizes != grads.sizes or dst.kinds != grads.kinds
                or dst.tensors[0].device != grads.tensors[0].device):
            raise ValueError("clip_grads: out must match the gradients' sizes, types and device")
    return ops.clip_grads(grads, dst, inf_norm, float(max_norm))


@ops.outside_graph
@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, *, sharded=(),
                    group=None) -> torch.Tensor:
    """Clip the parameters' .grad in place by their global norm; returns the norm.

    `sharded`: parameters of which each rank of `group` holds another part (the
    expert-parallel layer's packed experts): their share of the norm is summed over the group,
    while that of `parameters`, replicated on every rank, counts once.  With a `group` all its
    ranks make the call, those without sharded parameters too.  Parameters without a gradient
    are left out, and one that is listed twice counts once."""
    inf_norm = _inf(norm_type)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm must not be negative, got {max_norm!r}")
    parameters, own = (dict.fromkeys([p] if isinstance(p, torch.Tensor) else p)
                       for p in (parameters, sharded))
    whole = [p.grad for p in parameters if p.grad is not None and p not in own]
    parts = [p.grad for p in own if p.grad is not None]
    every = ops.GradList(whole + parts, "clip_grad_norm_")
    if group is None:
        if not every.tensors:
            return torch.zeros(())
        return ops.clip_grads(every, every, inf_norm, float(max_norm))
    # every rank takes part in the reduction, whatever it holds
    held = [*whole, *parts, *parameters, *own]
    device = held[0].device if held else "cuda" if torch.cuda.is_available() else "cpu"
    count = int(ops._lib.value("b200moe_grad_partials_count"))
    joined = torch.zeros(2, count, device=device, dtype=torch.float64)
    for row, grads in zip(joined, (whole, parts)):
        if grads:
            row.copy_(ops.grad_partials(ops.GradList(grads, "clip_grad_norm_"), inf_norm))
    if inf_norm:
        # The maximum of a reduction may pass over a NaN.  Partials are not negative, so their bits
        # without the sign, taken as integers, have their order, with a NaN above infinity.
        bits = joined[1].view(torch.int64).bitwise_and_(2 ** 63 - 1)
        dist.all_reduce(bits, op=dist.ReduceOp.MAX, group=group)
    else:
        dist.all_reduce(joined[1], group=group)
    return ops.grad_clip(every if every.tensors else None, inf_norm, joined.view(-1),
                         float(max_norm))
