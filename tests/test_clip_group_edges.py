"""The gradient clip over a process group at its edges, on CPU ranks (gloo, world 2).

As in test_step_ops_gloo.py, stand-ins compute on the CPU what the kernels return; these keep a
NaN wherever a tensor holds one, as the kernels do."""

import math
import os
import socket
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

COUNT = 592


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


class _Grads:
    def __init__(self, tensors, name):
        self.tensors = tensors


def _install_stand_ins():
    from spark_gpt_b200 import _lib, ops

    def grad_partials(grads, inf_norm):
        out = torch.zeros(COUNT, dtype=torch.float64)
        for i, t in enumerate(grads.tensors):
            v = t.double()
            j = i % COUNT
            out[j] = torch.maximum(out[j], v.abs().max()) if inf_norm else out[j] + v.square().sum()
        return out

    def grad_clip(grads, inf_norm, partials, max_norm):
        norm = float(partials.max() if inf_norm else partials.sum().sqrt())
        c = min(1.0, max_norm / (norm + 1e-6)) if math.isfinite(norm) else 1.0
        for t in grads.tensors if grads is not None else ():
            t.mul_(c)
        return torch.tensor(norm, dtype=torch.float32)

    def clip_grads(grads, out, inf_norm, max_norm):
        return grad_clip(grads, inf_norm, grad_partials(grads, inf_norm), max_norm)

    ops.GradList = _Grads
    ops.grad_partials = grad_partials
    ops.grad_clip = grad_clip
    ops.clip_grads = clip_grads
    _lib.value = lambda name, *a: COUNT


def _param(value, n):
    p = torch.nn.Parameter(torch.zeros(n))
    p.grad = torch.full((n,), float(value))
    return p


def _worker(rank, world, port, case, args, results):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=20))
    try:
        _install_stand_ins()
        results[rank] = case(rank, dist.group.WORLD, *args)
    finally:
        dist.destroy_process_group()


def _run(case, *args):
    results = mp.get_context("spawn").Manager().dict()
    mp.start_processes(_worker, args=(2, _free_port(), case, args, results), nprocs=2, join=True,
                       start_method="spawn")
    return results[0], results[1]


def _nonfinite(rank, group, values, norm_type):
    from spark_gpt_b200 import clip_grad_norm_
    shared, shard = _param(2.0, 4), _param(1.0 + rank, 9)
    if values[rank] is not None:
        shard.grad[3] = values[rank]
    before = shared.grad.clone(), shard.grad.clone()
    norm = float(clip_grad_norm_([shared], 0.1, norm_type, sharded=[shard], group=group))
    kept = all(torch.equal(a.nan_to_num(7.0), p.grad.nan_to_num(7.0))
               for a, p in zip(before, (shared, shard)))
    return norm, kept


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("values", [(math.nan, None), (None, math.nan), (-math.nan, math.inf),
                                    (math.inf, math.nan), (None, -math.inf)], ids=str)
def test_a_shard_that_is_not_finite_reaches_every_rank(values, norm_type):
    """Whichever rank holds a NaN, every rank's norm is NaN; without one an infinity is; and no
    gradient is scaled."""
    nan = any(v is not None and math.isnan(v) for v in values)
    for norm, kept in _run(_nonfinite, values, norm_type):
        assert math.isnan(norm) if nan else norm == math.inf
        assert kept


def _uneven(rank, group, nothing_at_all):
    from spark_gpt_b200 import clip_grad_norm_
    if rank == 1 and nothing_at_all:
        return float(clip_grad_norm_([], 1.0, group=group)), []
    shared = _param(2.0, 4)
    sharded = [_param(3.0, 9)] if rank == 0 else []
    norm = clip_grad_norm_((p for p in [shared, *sharded]), 1.0, sharded=sharded, group=group)
    return float(norm), [float(p.grad[0]) for p in [shared, *sharded]]


@pytest.mark.parametrize("nothing_at_all", [False, True])
def test_a_rank_without_sharded_parameters_takes_part(nothing_at_all):
    """Its norm and scale hold the other ranks' shards."""
    (norm, grads), (other, others) = _run(_uneven, nothing_at_all)
    want = math.sqrt(4 * 4.0 + 9 * 9.0)
    c = 1.0 / (want + 1e-6)
    assert math.isclose(norm, want, rel_tol=1e-6)
    assert math.isclose(grads[0], 2.0 * c, rel_tol=1e-6)
    assert math.isclose(grads[1], 3.0 * c, rel_tol=1e-6)
    if nothing_at_all:
        assert math.isclose(other, 9.0, rel_tol=1e-6)  # it replicates nothing: the shards alone
    else:
        assert math.isclose(other, want, rel_tol=1e-6)
        assert math.isclose(others[0], 2.0 * c, rel_tol=1e-6)


def _single(rank, group):
    from spark_gpt_b200 import clip_grad_norm_
    shard = _param(2.0 + rank, 4)
    norm = clip_grad_norm_([], 1.0, sharded=shard, group=group)
    return float(norm), float(shard.grad[0])


def test_a_single_sharded_parameter():
    """Given as itself, as `parameters` may be: not the list of its rows, which have no gradient."""
    want = math.sqrt(4 * 4.0 + 4 * 9.0)
    for rank, (norm, grad) in enumerate(_run(_single)):
        assert math.isclose(norm, want, rel_tol=1e-6)
        assert math.isclose(grad, (2.0 + rank) / (want + 1e-6), rel_tol=1e-6)
