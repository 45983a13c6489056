"""Tensor-level wrappers over the C ABI (include/b200moe.h).

Each function allocates its outputs through torch's caching allocator, passes
raw pointers plus torch's current CUDA stream to libb200moe.so, and returns
the outputs.  Shapes follow spark-gpt's MoE path (train.py:2134-2334).
"""

from __future__ import annotations

import ctypes
from array import array
from contextlib import contextmanager
from dataclasses import dataclass
from functools import lru_cache

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib

# --------------------------------------------------------------------------- #
# launch accounting and optional per-op CUDA-event timing (used by bench.py)
# --------------------------------------------------------------------------- #
LAUNCHES = {"count": 0}
_timing: dict[str, list] | None = None


def set_timing(names):
    """Record CUDA events around the named ops (None disables)."""
    global _timing
    _timing = None if names is None else {n: [] for n in names}
    return _timing


@contextmanager
def timed(name: str):
    """CUDA events on the current stream around a block (e.g. a collective)."""
    if _timing is not None and name in _timing:
        s = torch.cuda.Event(enable_timing=True)
        e = torch.cuda.Event(enable_timing=True)
        s.record()
        yield
        e.record()
        _timing[name].append((s, e))
    else:
        yield


@contextmanager
def persistent_sm_limit(sms: int):
    """Persistent kernels enqueued inside the block use at most `sms` SMs
    (0 = all), leaving the rest to a collective running beside them."""
    prev = int(_lib.value("b200moe_set_persistent_sm_limit", int(sms)))
    try:
        yield
    finally:
        _lib.value("b200moe_set_persistent_sm_limit", prev)


@contextmanager
def transfer_sm_limit(sms: int):
    """Peer-memory transfer kernels enqueued inside the block launch at most 8
    blocks per SM of `sms` SMs (0 = all), leaving the other SMs to the
    kernels of the stream they run beside."""
    prev = int(_lib.value("b200moe_set_transfer_sm_limit", int(sms)))
    try:
        yield
    finally:
        _lib.value("b200moe_set_transfer_sm_limit", prev)


def _launch(name: str, kernels: int, fn, *args):
    LAUNCHES["count"] += kernels
    if _timing is not None and name in _timing:
        s = torch.cuda.Event(enable_timing=True)
        e = torch.cuda.Event(enable_timing=True)
        s.record()
        _lib.call(fn, *args)
        e.record()
        _timing[name].append((s, e))
    else:
        _lib.call(fn, *args)


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _s(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _check(t: torch.Tensor, dtype, name):
    if not t.is_cuda:
        raise RuntimeError(f"{name}: the B200 MoE kernels need CUDA tensors (no CPU path)")
    if t.dtype != dtype:
        raise RuntimeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name}: expected a contiguous tensor")


BF16 = torch.bfloat16


def padded_rows(routed_rows: int, num_experts: int) -> int:
    return int(_lib.value("b200moe_padded_rows", routed_rows, num_experts))


def router_width(num_experts: int) -> int:
    return int(_lib.value("b200moe_router_width", num_experts))


# --------------------------------------------------------------------------- #
# weights
# --------------------------------------------------------------------------- #
def cast_bf16(w: torch.Tensor, rows_out: int | None = None) -> torch.Tensor:
    """bf16 compute copy of an fp32 master (rows beyond w.shape[0] zero)."""
    if w.dtype == BF16 and rows_out in (None, w.shape[0]):
        return w.contiguous()
    w = w.detach().float().contiguous()
    rows = w.shape[0]
    cols = w[0].numel() if rows else 0
    rows_out = rows if rows_out is None else rows_out
    out = torch.empty((rows_out, *w.shape[1:]), device=w.device, dtype=BF16)
    _launch("cast", 1, "b200moe_cast_f32_to_bf16", _p(w), rows, cols, rows_out, _p(out), _s(w))
    return out


# --------------------------------------------------------------------------- #
# router (train.py:2144-2158)
# --------------------------------------------------------------------------- #
def router_logits(x: torch.Tensor, w_router: torch.Tensor) -> torch.Tensor:
    _check(x, BF16, "router_logits x")
    _check(w_router, BF16, "router_logits w")
    T, H = x.shape
    W = w_router.shape[0]
    out = torch.empty(T, W, device=x.device, dtype=BF16)
    if T:
        _launch("router_logits", 1, "b200moe_router_logits", _p(x), _p(w_router), T, H, W,
                _p(out), _s(x))
    return out


def router_topk(logits: torch.Tensor, num_experts: int, top_k: int, norm: bool):
    """logits (T, ld) bf16 or fp32 (first num_experts columns used)."""
    if logits.dtype not in (BF16, torch.float32):
        raise RuntimeError("router_topk: logits must be bf16 or fp32")
    if logits.stride(1) != 1:
        raise RuntimeError("router_topk: logits rows must be contiguous")
    T = logits.shape[0]
    sel = torch.empty(T, top_k, device=logits.device, dtype=torch.int64)
    w = torch.empty(T, top_k, device=logits.device, dtype=BF16)
    if T:
        _launch("router_topk", 1, "b200moe_router_topk_fwd", _p(logits),
                int(logits.dtype == torch.float32), logits.stride(0), T, num_experts, top_k,
                int(norm), _p(sel), _p(w), _s(logits))
    return sel, w


def router_topk_bwd(logits, selected, d_weights, d_extra, num_experts, top_k, norm):
    T, ld = logits.shape[0], logits.stride(0)
    out = torch.empty(T, ld, device=logits.device, dtype=BF16)
    if T:
        _launch("router_topk_bwd", 1, "b200moe_router_topk_bwd", _p(logits), ld, _p(selected),
                _p(d_weights), _p(d_extra), T, num_experts, top_k, int(norm), _p(out),
                _s(logits))
    return out


def router_dgrad(d_logits: torch.Tensor, w_router: torch.Tensor) -> torch.Tensor:
    T, W = d_logits.shape
    H = w_router.shape[1]
    out = torch.empty(T, H, device=d_logits.device, dtype=BF16)
    if T:
        _launch("router_dgrad", 1, "b200moe_router_dgrad", _p(d_logits), _p(w_router), T, H, W,
                _p(out), _s(d_logits))
    return out


def router_wgrad(x, d_logits, num_experts, out=None, accumulate=False):
    T, H = x.shape
    W = d_logits.shape[1]
    if out is None:
        out = torch.empty(num_experts, H, device=x.device, dtype=torch.float32)
        accumulate = False
    if T:
        nbytes = int(_lib.value("b200moe_router_wgrad_scratch_bytes", T, H, num_experts))
        scratch = torch.empty(max(nbytes, 16), device=x.device, dtype=torch.uint8)
        _launch("router_wgrad", 2, "b200moe_router_wgrad", _p(x), _p(d_logits), T, H,
                num_experts, W, _p(out), int(accumulate), _p(scratch), nbytes, _s(x))
    elif not accumulate:
        out.zero_()
    return out


# --------------------------------------------------------------------------- #
# dispatch (train.py:2271-2290)
# --------------------------------------------------------------------------- #
@dataclass
class Dispatch:
    counts: torch.Tensor       # (E,) int32
    offsets: torch.Tensor      # (E,) int32 inclusive cumsum
    pad_offsets: torch.Tensor  # (E+1,) int32 padded starts; [E] = padded total
    row_flat: torch.Tensor     # (Rcap,) int32 padded row -> flat slot, -1 padding
    inv_pad: torch.Tensor      # (R,) int32 flat slot -> padded row
    tile_expert: torch.Tensor  # (Rcap/128,) int32
    rows_cap: int
    num_tokens: int
    top_k: int
    num_experts: int
    partial: bool = False      # some slots carry no expert (id -1: no row, inv_pad -1)


def dispatch(selected: torch.Tensor, num_experts: int, routed_slots: int | None = None,
             partial: bool = False) -> Dispatch:
    """partial: negative ids may occur and mark slots without an expert (no row,
    inv_pad -1; the row reductions then skip them).  routed_slots, when given,
    is the number of non-negative ids and sizes the padded-row buffers."""
    _check(selected, torch.int64, "dispatch selected")
    T, k = selected.shape
    R = T * k
    dev = selected.device
    cap = padded_rows(R if routed_slots is None else routed_slots, num_experts)
    i32 = dict(device=dev, dtype=torch.int32)
    if R == 0:  # no slots: every expert empty, every row padding (nothing to launch)
        z = lambda n: torch.zeros(n, **i32)  # noqa: E731
        return Dispatch(z(num_experts), z(num_experts), z(num_experts + 1),
                        torch.full((cap,), -1, **i32), z(0), z(cap // 128), cap, T, k,
                        num_experts, partial or routed_slots is not None)
    counts = torch.empty(num_experts, **i32)
    offsets = torch.empty(num_experts, **i32)
    pad = torch.empty(num_experts + 1, **i32)
    row_flat = torch.empty(cap, **i32)
    inv = torch.empty(max(R, 1), **i32)
    tiles = torch.empty(cap // 128, **i32)
    nbytes = int(_lib.value("b200moe_dispatch_scratch_bytes", T, k, num_experts))
    scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    _launch("dispatch", 3, "b200moe_dispatch", _p(selected), T, k, num_experts, _p(counts),
            _p(offsets), _p(pad), _p(row_flat), _p(inv), _p(tiles), _p(scratch), nbytes,
            _s(selected))
    return Dispatch(counts, offsets, pad, row_flat, inv[:R], tiles, cap, T, k, num_experts,
                    partial or routed_slots is not None)


# --------------------------------------------------------------------------- #
# gather / combine (train.py:2195-2241)
# --------------------------------------------------------------------------- #
def _rows_out(out, rows: int, cols: int, like: torch.Tensor, name: str) -> torch.Tensor:
    """A caller's (rows, cols) bf16 destination (checked), or a new one."""
    if out is None:
        return torch.empty(rows, cols, device=like.device, dtype=BF16)
    _check(out, BF16, name)
    if tuple(out.shape) != (rows, cols):
        raise RuntimeError(f"{name}: expected shape {(rows, cols)}, got {tuple(out.shape)}")
    return out


def gather_rows(x: torch.Tensor, d: Dispatch, out=None) -> torch.Tensor:
    """out: an optional contiguous (rows_cap, H) bf16 destination."""
    _check(x, BF16, "gather_rows x")
    H = x.shape[1]
    xs = _rows_out(out, d.rows_cap, H, x, "gather_rows out")
    if d.num_tokens == 0:  # only padding rows
        return xs.zero_()
    _launch("gather", 1, "b200moe_gather_rows", _p(x), _p(d.row_flat),
            _p(d.inv_pad) if d.inv_pad.numel() else None, _p(d.pad_offsets), d.num_tokens,
            d.num_experts, d.top_k, H, d.rows_cap, _p(xs), _s(x))
    return xs


def gather_rows_bwd(dxs, d: Dispatch, addend=None, token_major=False, out=None) -> torch.Tensor:
    """dx[t] = sum_s dxs[row of slot t*k+s] (+ addend); token_major: row t*k+s.
    out: an optional contiguous (T, H) bf16 destination."""
    H = dxs.shape[1]
    if out is None:
        dx = torch.empty(d.num_tokens, H, device=dxs.device, dtype=BF16)
    else:
        _check(out, BF16, "gather_rows_bwd out")
        dx = out
    if d.num_tokens:
        _launch("gather_bwd", 1, "b200moe_gather_rows_bwd", _p(dxs),
                None if token_major else _p(d.inv_pad), _p(addend), d.num_tokens, d.top_k, H,
                int(d.partial), _p(dx), _s(dxs))
    return dx


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float):
    """The reference's RMSNorm (train.py:162-170) on bf16 rows: (x_n bf16, r fp32 per row)."""
    _check(x, BF16, "rmsnorm x")
    T, H = x.shape
    wf = w.detach().float().contiguous()
    x_n = torch.empty_like(x)
    rstd = torch.empty(T, device=x.device, dtype=torch.float32)
    if T:
        _launch("rmsnorm", 1, "b200moe_rmsnorm_fwd", _p(x), _p(wf), T, H, ctypes.c_float(eps),
                _p(x_n), _p(rstd), _s(x))
    return x_n, rstd


def gather_rows_bwd_rmsnorm(dxs, d: Dispatch, addend, x, w, rstd, token_major=False):
    """The gather backward (dxs rows summed per token + addend) with the
    RMSNorm backward folded in: (d x (T, H) bf16, d w (H,) fp32)."""
    H = dxs.shape[1]
    dev = dxs.device
    dx = torch.empty(d.num_tokens, H, device=dev, dtype=BF16)
    dw = torch.empty(H, device=dev, dtype=torch.float32)
    nbytes = int(_lib.value("b200moe_gather_rows_bwd_rmsnorm_scratch_bytes", d.num_tokens, H))
    scratch = torch.empty(max(nbytes, 16), device=dev, dtype=torch.uint8)
    _launch("gather_bwd", 2, "b200moe_gather_rows_bwd_rmsnorm", _p(dxs),
            None if token_major else _p(d.inv_pad), _p(addend), _p(x), _p(w), _p(rstd),
            d.num_tokens, d.top_k, H, int(d.partial), _p(dx), _p(dw), _p(scratch), nbytes,
            _s(dxs))
    return dx, dw


def combine(y, d: Dispatch, weights, token_major=False) -> torch.Tensor:
    _check(weights, BF16, "combine weights")
    H = y.shape[1]
    out = torch.empty(d.num_tokens, H, device=y.device, dtype=BF16)
    if d.num_tokens:
        _launch("combine", 1, "b200moe_combine_fwd", _p(y),
                None if token_major else _p(d.inv_pad), _p(weights), d.num_tokens, d.top_k, H,
                int(d.partial), _p(out), _s(y))
    return out


def combine_bwd(d_out, y, d: Dispatch, weights, token_major=False, out=None):
    """-> (dy (rows_cap, H) bf16, d_weights (T, k) fp32); out: an optional
    contiguous destination for dy."""
    _check(d_out, BF16, "combine_bwd d_out")
    H = y.shape[1]
    dy = _rows_out(out, d.rows_cap, H, y, "combine_bwd out")
    if d.num_tokens == 0:  # only padding rows, no routing weights
        return dy.zero_(), torch.zeros(0, d.top_k, device=y.device, dtype=torch.float32)
    dw = torch.empty(d.num_tokens, d.top_k, device=y.device, dtype=torch.float32)
    _launch("combine_bwd", 2 if token_major else 1, "b200moe_combine_bwd", _p(d_out), _p(y),
            _p(d.row_flat), _p(d.inv_pad), _p(d.pad_offsets), _p(weights), d.num_experts,
            d.num_tokens, d.top_k, H, d.rows_cap, int(token_major), _p(dy), _p(dw), _s(y))
    return dy, dw


# --------------------------------------------------------------------------- #
# expert products (train.py:1625-2090)
# --------------------------------------------------------------------------- #
def gate_up_fwd(xs, w_gu, d: Dispatch, out_h=None):
    """-> (gu, h); out_h: an optional contiguous (rows_cap, I) bf16 destination."""
    E, two_i, H = w_gu.shape
    I = two_i // 2
    gu = torch.empty(d.rows_cap, two_i, device=xs.device, dtype=BF16)
    h = _rows_out(out_h, d.rows_cap, I, xs, "gate_up_fwd out_h")
    _launch("gate_up_fwd", 1, "b200moe_expert_gate_up_fwd", _p(xs), _p(w_gu), _p(d.tile_expert),
            _p(d.pad_offsets), d.rows_cap, E, H, I, _p(gu), _p(h), _s(xs))
    return gu, h


def down_fwd(h, w_d, d: Dispatch, token_major=False):
    """y = h W_d[e]^T; token_major: (T*k, H) with slot t*k+s in row t*k+s."""
    E, H, I = w_d.shape
    rows = d.num_tokens * d.top_k if token_major else d.rows_cap
    y = torch.empty(max(rows, 1), H, device=h.device, dtype=BF16)
    _launch("down_fwd", 1, "b200moe_expert_down_fwd", _p(h), _p(w_d), _p(d.tile_expert),
            _p(d.pad_offsets), _p(d.row_flat) if token_major else None, d.rows_cap, E, H, I,
            _p(y), _s(h))
    return y


def down_dgrad_swiglu(dy, w_d, gu, d: Dispatch, out=None):
    """d_gu (rows_cap, 2I) bf16; out: an optional contiguous destination."""
    E, H, I = w_d.shape
    d_gu = _rows_out(out, d.rows_cap, 2 * I, dy, "down_dgrad_swiglu out")
    _launch("down_dgrad", 1, "b200moe_expert_down_dgrad_swiglu", _p(dy), _p(w_d), _p(gu),
            _p(d.tile_expert), _p(d.pad_offsets), d.rows_cap, E, H, I, _p(d_gu), _s(dy))
    return d_gu


def gate_up_dgrad(d_gu, w_gu, d: Dispatch, token_major=False):
    """dxs = d_gu W_gu[e]; token_major: (T*k, H) with slot t*k+s in row t*k+s."""
    E, two_i, H = w_gu.shape
    rows = d.num_tokens * d.top_k if token_major else d.rows_cap
    dxs = torch.empty(max(rows, 1), H, device=d_gu.device, dtype=BF16)
    _launch("gate_up_dgrad", 1, "b200moe_expert_gate_up_dgrad", _p(d_gu), _p(w_gu),
            _p(d.tile_expert), _p(d.pad_offsets), _p(d.row_flat) if token_major else None,
            d.rows_cap, E, H, two_i // 2, _p(dxs), _s(d_gu))
    return dxs


def wgrad(a, b, d: Dispatch, name="wgrad", out=None, accumulate=False):
    """(E, M, N) fp32: a_e^T b_e over the padded rows of each expert."""
    M, N = a.shape[1], b.shape[1]
    if out is None:
        out = torch.empty(d.num_experts, M, N, device=a.device, dtype=torch.float32)
        accumulate = False
    _launch(name, 1, "b200moe_expert_wgrad", _p(a), M, _p(b), N, _p(d.pad_offsets),
            d.num_experts, d.rows_cap, _p(out), int(accumulate), _s(a))
    return out


def wgrad_segments(a, b, seg_offsets, num_experts, name="wgrad", out=None, accumulate=False):
    """(E, M, N) fp32: a_e^T b_e where expert e's rows are the union over
    segments s of [seg_offsets[s, e], seg_offsets[s, e+1]) of a and b
    (rows_total, M) / (rows_total, N) bf16; seg_offsets (S, E+1) int32."""
    M, N = a.shape[1], b.shape[1]
    _check(a, BF16, f"{name} a")
    _check(b, BF16, f"{name} b")
    if a.shape[0] != b.shape[0]:
        raise RuntimeError(f"{name}: a and b must have the same rows")
    _check(seg_offsets, torch.int32, f"{name} seg_offsets")
    if seg_offsets.dim() != 2 or seg_offsets.shape[1] != num_experts + 1:
        raise RuntimeError(f"{name}: seg_offsets must be (segments, E+1)")
    if out is None:
        out = torch.empty(num_experts, M, N, device=a.device, dtype=torch.float32)
        accumulate = False
    _launch(name, 1, "b200moe_expert_wgrad_segments", _p(a), M, _p(b), N, _p(seg_offsets),
            seg_offsets.shape[0], num_experts, a.shape[0], _p(out), int(accumulate), _s(a))
    return out


# --------------------------------------------------------------------------- #
# fp8 expert path (spark-gpt --fp8-mlp, train.py:1301-1604)
# --------------------------------------------------------------------------- #
E4M3 = torch.float8_e4m3fn
E5M2 = torch.float8_e5m2
_FP8_FMT = {E4M3: 0, E5M2: 1}


def _check_fp8(t: torch.Tensor, name, dtypes=(E4M3, E5M2)):
    if not t.is_cuda:
        raise RuntimeError(f"{name}: the B200 MoE kernels need CUDA tensors (no CPU path)")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name}: expected one of {dtypes}, got {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name}: expected a contiguous tensor")


def _check_scales(scale, amax=None):
    _check(scale, torch.float32, "fp8 scale")
    if scale.numel() < 5:
        raise RuntimeError("fp8 scale: expected the five per-site scales")
    if amax is not None:
        _check(amax, torch.float32, "fp8 amax")
        if amax.numel() < 5:
            raise RuntimeError("fp8 amax: expected the five amax slots")


def fp8_quantize_experts(w: torch.Tensor):
    """(e4m3 copy of w * q_e, q (E,) fp32) of fp32 (E, rows, cols) master
    weights, q_e = 2^floor(log2(448 / max|w_e|)) (train.py:1536-1540)."""
    w = w.detach().float().contiguous()
    E = w.shape[0]
    per = w[0].numel() if E else 0
    w8 = torch.empty(w.shape, device=w.device, dtype=E4M3)
    q = torch.empty(E, device=w.device, dtype=torch.float32)
    if E and per:
        nbytes = int(_lib.value("b200moe_fp8_quantize_experts_scratch_bytes", E))
        scratch = torch.empty(nbytes, device=w.device, dtype=torch.uint8)
        _launch("fp8_quantize", 3, "b200moe_fp8_quantize_experts", _p(w), E, per, _p(w8), _p(q),
                _p(scratch), nbytes, _s(w))
    return w8, q


def fp8_gather_quant(x: torch.Tensor, d: Dispatch, scale, amax) -> torch.Tensor:
    """x8 (Rcap, H) e4m3 = e4m3(x[token] * scale[0]), padding rows zero; amax[0] raised."""
    _check(x, BF16, "fp8_gather_quant x")
    _check_scales(scale, amax)
    H = x.shape[1]
    x8 = torch.empty(d.rows_cap, H, device=x.device, dtype=E4M3)
    if d.num_tokens == 0:
        return x8.zero_()
    _launch("gather", 1, "b200moe_fp8_gather_quant", _p(x), _p(d.row_flat), _p(d.inv_pad),
            _p(d.pad_offsets), d.num_tokens, d.num_experts, d.top_k, H, d.rows_cap, _p(scale),
            _p(amax), _p(x8), _s(x))
    return x8


def fp8_quantize_rows(src: torch.Tensor, scale_slot: torch.Tensor, amax_slot: torch.Tensor,
                      dtype=E5M2, d: Dispatch | None = None) -> torch.Tensor:
    """fp8(src * scale_slot[0]) of a bf16 matrix, amax_slot[0] raised; with a
    Dispatch, only the rows below its padded total (the rest of a padded-row
    buffer holds no data and is left unwritten)."""
    _check(src, BF16, "fp8_quantize_rows src")
    dst = torch.empty(src.shape, device=src.device, dtype=dtype)
    rows, cols = src.shape
    total = None if d is None else d.pad_offsets[d.num_experts:]
    _launch("fp8_quantize_rows", 1, "b200moe_fp8_quantize_rows", _p(src), rows, cols, _p(total),
            _p(scale_slot), _p(amax_slot), _FP8_FMT[dtype], _p(dst), _s(src))
    return dst


def fp8_combine_bwd(d_out, y, d: Dispatch, weights, scale_slot, amax_slot):
    """combine_bwd that also returns dy8 = e5m2(dy * scale_slot[0]) (padding
    rows zero) and raises amax_slot[0] with max|dy| (one pass over dy)."""
    _check(d_out, BF16, "fp8_combine_bwd d_out")
    _check(weights, BF16, "fp8_combine_bwd weights")
    H = y.shape[1]
    if d.num_tokens == 0:
        return (torch.zeros(d.rows_cap, H, device=y.device, dtype=BF16),
                torch.zeros(0, d.top_k, device=y.device, dtype=torch.float32),
                torch.zeros(d.rows_cap, H, device=y.device, dtype=E5M2))
    dy = torch.empty(d.rows_cap, H, device=y.device, dtype=BF16)
    dy8 = torch.empty(d.rows_cap, H, device=y.device, dtype=E5M2)
    dw = torch.empty(d.num_tokens, d.top_k, device=y.device, dtype=torch.float32)
    _launch("combine_bwd", 1, "b200moe_fp8_combine_bwd", _p(d_out), _p(y), _p(d.row_flat),
            _p(d.inv_pad), _p(d.pad_offsets), _p(weights), d.num_experts, d.num_tokens,
            d.top_k, H, d.rows_cap, _p(scale_slot), _p(amax_slot), _p(dy), _p(dw), _p(dy8),
            _s(y))
    return dy, dw, dy8


def fp8_gate_up_fwd(x8, w8_gu, q_gu, d: Dispatch, scale, amax):
    """gu8 (Rcap, 2I), h8 (Rcap, I) e4m3 (train.py:1317-1354)."""
    _check_fp8(x8, "fp8_gate_up_fwd x8", (E4M3,))
    _check_fp8(w8_gu, "fp8_gate_up_fwd w8", (E4M3,))
    _check_scales(scale, amax)
    E, two_i, H = w8_gu.shape
    I = two_i // 2
    gu8 = torch.empty(d.rows_cap, two_i, device=x8.device, dtype=E4M3)
    h8 = torch.empty(d.rows_cap, I, device=x8.device, dtype=E4M3)
    _launch("gate_up_fwd", 1, "b200moe_fp8_expert_gate_up_fwd", _p(x8), _p(w8_gu), _p(q_gu),
            _p(d.tile_expert), _p(d.pad_offsets), d.rows_cap, E, H, I, _p(scale), _p(amax),
            _p(gu8), _p(h8), _s(x8))
    return gu8, h8


def fp8_down_fwd(h8, wd8, q_d, d: Dispatch, scale):
    """y (Rcap, H) bf16 = h8 . W8_d[e]^T / (scale[2] q_d[e]) (train.py:1357-1379)."""
    _check_fp8(h8, "fp8_down_fwd h8", (E4M3,))
    _check_fp8(wd8, "fp8_down_fwd w8", (E4M3,))
    _check_scales(scale)
    E, H, I = wd8.shape
    y = torch.empty(d.rows_cap, H, device=h8.device, dtype=BF16)
    _launch("down_fwd", 1, "b200moe_fp8_expert_down_fwd", _p(h8), _p(wd8), _p(q_d),
            _p(d.tile_expert), _p(d.pad_offsets), d.rows_cap, E, H, I, _p(scale), _p(y), _s(h8))
    return y


def fp8_down_dgrad_swiglu(dy, w_d, gu8, d: Dispatch, scale, amax):
    """d_gu8 (Rcap, 2I) e5m2 from bf16 dy and W_d (train.py:1382-1423)."""
    _check(dy, BF16, "fp8_down_dgrad dy")
    _check(w_d, BF16, "fp8_down_dgrad w")
    _check_fp8(gu8, "fp8_down_dgrad gu8", (E4M3,))
    _check_scales(scale, amax)
    E, H, I = w_d.shape
    d_gu8 = torch.empty(d.rows_cap, 2 * I, device=dy.device, dtype=E5M2)
    _launch("down_dgrad", 1, "b200moe_fp8_expert_down_dgrad_swiglu", _p(dy), _p(w_d), _p(gu8),
            _p(d.tile_expert), _p(d.pad_offsets), d.rows_cap, E, H, I, _p(scale), _p(amax),
            _p(d_gu8), _s(dy))
    return d_gu8


def fp8_gate_up_dgrad(d_gu8, w8_gu, q_gu, d: Dispatch, scale):
    """dxs (Rcap, H) bf16 = d_gu8 . W8_gu[e] / (scale[3] q_gu[e]) (train.py:1426-1448)."""
    _check_fp8(d_gu8, "fp8_gate_up_dgrad d_gu8", (E5M2,))
    _check_fp8(w8_gu, "fp8_gate_up_dgrad w8", (E4M3,))
    _check_scales(scale)
    E, two_i, H = w8_gu.shape
    dxs = torch.empty(d.rows_cap, H, device=d_gu8.device, dtype=BF16)
    _launch("gate_up_dgrad", 1, "b200moe_fp8_expert_gate_up_dgrad", _p(d_gu8), _p(w8_gu),
            _p(q_gu), _p(d.tile_expert), _p(d.pad_offsets), d.rows_cap, E, H, two_i // 2,
            _p(scale), _p(dxs), _s(d_gu8))
    return dxs


def fp8_wgrad(a8, b8, d: Dispatch, scale_a, scale_b, name="wgrad", out=None, accumulate=False):
    """(E, M, N) fp32 (+)= a8_e^T b8_e / (scale_a[0] scale_b[0]) over the padded
    rows of each expert (train.py:1451-1478, :1504-1530)."""
    _check_fp8(a8, f"{name} a8")
    _check_fp8(b8, f"{name} b8", (E4M3,))
    M, N = a8.shape[1], b8.shape[1]
    if out is None:
        out = torch.empty(d.num_experts, M, N, device=a8.device, dtype=torch.float32)
        accumulate = False
    _launch(name, 1, "b200moe_fp8_expert_wgrad", _p(a8), _FP8_FMT[a8.dtype], M, _p(b8), N,
            _p(d.pad_offsets), d.num_experts, d.rows_cap, _p(scale_a), _p(scale_b), _p(out),
            int(accumulate), _s(a8))
    return out


# --------------------------------------------------------------------------- #
# expert products with the row gather / combine backward fused in
# --------------------------------------------------------------------------- #
def gate_up_fwd_gather(x, w_gu, d: Dispatch):
    """gate_up fwd reading xs[p] = x[row_flat[p]/k] in the GEMM's loads."""
    _check(x, BF16, "gate_up_fwd_gather x")
    E, two_i, H = w_gu.shape
    I = two_i // 2
    gu = torch.empty(d.rows_cap, two_i, device=x.device, dtype=BF16)
    h = torch.empty(d.rows_cap, I, device=x.device, dtype=BF16)
    _launch("gate_up_fwd", 1, "b200moe_expert_gate_up_fwd_gather", _p(x), _p(d.row_flat),
            d.num_tokens, d.top_k, _p(w_gu), _p(d.tile_expert), _p(d.pad_offsets), d.rows_cap,
            E, H, I, _p(gu), _p(h), _s(x))
    return gu, h


def down_dgrad_combine(d_out, weights, w_d, gu, h, d: Dispatch):
    """Combine backward + down dgrad + SwiGLU backward -> (d_gu, w*h, d_weights (T,k))."""
    _check(d_out, BF16, "down_dgrad_combine d_out")
    _check(weights, BF16, "down_dgrad_combine weights")
    E, H, I = w_d.shape
    dev = d_out.device
    d_gu = torch.empty(d.rows_cap, 2 * I, device=dev, dtype=BF16)
    hw = torch.empty(d.rows_cap, I, device=dev, dtype=BF16)
    d_w = torch.empty(d.num_tokens, d.top_k, device=dev, dtype=torch.float32)
    nbytes = int(_lib.value("b200moe_down_dgrad_combine_scratch_bytes", d.rows_cap, I))
    scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    _launch("down_dgrad", 2, "b200moe_expert_down_dgrad_combine", _p(d_out), _p(d.row_flat),
            _p(weights), d.num_tokens, d.top_k, _p(w_d), _p(gu), _p(h), _p(d.tile_expert),
            _p(d.pad_offsets), d.rows_cap, E, H, I, _p(d_gu), _p(hw), _p(d_w), _p(scratch),
            nbytes, _s(d_out))
    return d_gu, hw, d_w


def wgrad_gather_b(a, x, d: Dispatch, name="wgrad", out=None, accumulate=False):
    """(E, M, N) fp32: a_e^T x[tokens of expert e]."""
    M, N = a.shape[1], x.shape[1]
    if out is None:
        out = torch.empty(d.num_experts, M, N, device=a.device, dtype=torch.float32)
        accumulate = False
    _launch(name, 1, "b200moe_expert_wgrad_gather_b", _p(a), M, _p(x), N, _p(d.row_flat),
            d.num_tokens, d.top_k, _p(d.pad_offsets), d.num_experts, d.rows_cap, _p(out),
            int(accumulate), _s(a))
    return out


def wgrad_gather_a(src, b, d: Dispatch, name="wgrad", out=None, accumulate=False):
    """(E, M, N) fp32: src[tokens of expert e]^T b_e."""
    M, N = src.shape[1], b.shape[1]
    if out is None:
        out = torch.empty(d.num_experts, M, N, device=b.device, dtype=torch.float32)
        accumulate = False
    _launch(name, 1, "b200moe_expert_wgrad_gather_a", _p(src), M, _p(d.row_flat), d.num_tokens,
            d.top_k, _p(b), N, _p(d.pad_offsets), d.num_experts, d.rows_cap, _p(out),
            int(accumulate), _s(b))
    return out


# --------------------------------------------------------------------------- #
# expert parallel: send plan, slot words, routing-weight gradient
# --------------------------------------------------------------------------- #
def ep_route(selected: torch.Tensor, experts_per_rank: int, ranks: int):
    """dest (T, P) int64 (r or -1 per destination rank) and the routed slots
    per destination rank (P,) int32."""
    _check(selected, torch.int64, "ep_route selected")
    T, k = selected.shape
    dest = torch.empty(T, ranks, device=selected.device, dtype=torch.int64)
    slots = torch.empty(ranks, device=selected.device, dtype=torch.int32)
    if T == 0:
        return dest, slots.zero_()
    _launch("ep_route", 1, "b200moe_ep_route", _p(selected), T, k, experts_per_rank, ranks,
            _p(dest), _p(slots), _s(selected))
    return dest, slots


def ep_pack(selected, weights, send: Dispatch, experts_per_rank: int) -> torch.Tensor:
    """(send.rows_cap, k) int32 slot words of the send rows."""
    _check(weights, BF16, "ep_pack weights")
    k = selected.shape[1]
    if selected.shape[0] == 0:  # no rows to send: every slot word says "no expert"
        return torch.full((send.rows_cap, k), 0xFFFF, device=selected.device, dtype=torch.int32)
    meta = torch.empty(send.rows_cap, k, device=selected.device, dtype=torch.int32)
    _launch("ep_pack", 1, "b200moe_ep_pack", _p(selected), _p(weights), _p(send.row_flat),
            _p(send.pad_offsets), send.rows_cap, k, experts_per_rank, send.num_experts,
            _p(meta), _s(selected))
    return meta


def ep_unpack(meta: torch.Tensor):
    """slot words (n, k) -> local expert ids (n, k) int64 (-1: foreign) and bf16 weights."""
    _check(meta, torch.int32, "ep_unpack meta")
    n, k = meta.shape
    sel = torch.empty(n, k, device=meta.device, dtype=torch.int64)
    w = torch.empty(n, k, device=meta.device, dtype=BF16)
    if n:
        _launch("ep_unpack", 1, "b200moe_ep_unpack", _p(meta), n, k, _p(sel), _p(w), _s(meta))
    return sel, w


def ep_p2p_plan(counts: torch.Tensor, me: int, ranks: int) -> torch.Tensor:
    """counts (P, ld) int32 gathered on every rank -> this rank's plan (2 + 4P ints)."""
    plan = torch.empty(2 + 4 * ranks, device=counts.device, dtype=torch.int32)
    _launch("ep_p2p_plan", 1, "b200moe_ep_p2p_plan", _p(counts), counts.stride(0), me, ranks,
            _p(plan), _s(counts))
    return plan


def ep_p2p_send(src, send: Dispatch, plan, peer_rows, selected=None, weights=None,
                experts_per_rank: int = 1, peer_meta=None):
    """Store each token's row (and slot words) into the owners' receive buffers."""
    _check(src, BF16, "ep_p2p_send src")
    T, H = src.shape
    if T == 0:
        return
    k = selected.shape[1] if selected is not None else 0
    _launch("ep_p2p_send", 1, "b200moe_ep_p2p_send", _p(src), _p(send.inv_pad),
            _p(send.pad_offsets), _p(plan), _p(peer_rows), T, H, send.num_experts,
            _p(selected), _p(weights), k, experts_per_rank, _p(peer_meta), _s(src))


def ep_p2p_send_part(src, send: Dispatch, plan, peer_rows, me: int, dest_mode: int,
                     selected=None, weights=None, experts_per_rank: int = 1, peer_meta=None):
    """ep_p2p_send restricted to this rank's own rows (dest_mode 1) or to the
    other ranks' rows (dest_mode 2)."""
    _check(src, BF16, "ep_p2p_send_part src")
    T, H = src.shape
    if T == 0:
        return
    k = selected.shape[1] if selected is not None else 0
    _launch("ep_p2p_send", 1, "b200moe_ep_p2p_send_part", _p(src), _p(send.inv_pad),
            _p(send.pad_offsets), _p(plan), _p(peer_rows), T, H, send.num_experts,
            _p(selected), _p(weights), k, experts_per_rank, _p(peer_meta), me, dest_mode,
            _s(src))


def ep_p2p_reduce_return_src(rows, d: Dispatch, plan, peer_rows, ranks: int, src: int,
                             weights=None, dw_rows=None, peer_dw=None):
    """Owner side, one source's chunk: each of its rows' local-slot sum stored
    into the source's back rows (and the routing-weight gradients into its back dw)."""
    H = rows.shape[1]
    _launch("ep_p2p_reduce_return", 1, "b200moe_ep_p2p_reduce_return_src", _p(rows),
            _p(d.inv_pad), _p(weights), d.top_k, _p(dw_rows), _p(plan), _p(peer_rows),
            _p(peer_dw), d.num_tokens, src, H, ranks, _s(rows))


def ep_signal(peer_flags, phase: int, me: int, ranks: int, epoch: int, dest: int = -1):
    _launch("ep_signal", 1, "b200moe_ep_signal", _p(peer_flags), phase, me, ranks, dest,
            ctypes.c_ulonglong(epoch), _s(peer_flags))


def ep_wait(my_flags, phase: int, ranks: int, epoch: int, src: int = -1):
    _launch("ep_wait", 1, "b200moe_ep_wait", _p(my_flags), phase, src, ranks,
            ctypes.c_ulonglong(epoch), _s(my_flags))


def ep_p2p_return(rows, plan, peer_rows, ranks: int, dw_rows=None, peer_dw=None):
    """Store the owner's result rows (and routing-weight gradients) into the sources' back buffers."""
    _check(rows, BF16, "ep_p2p_return rows")
    n, H = rows.shape
    k = dw_rows.shape[1] if dw_rows is not None else 0
    if n == 0:
        return
    _launch("ep_p2p_return", 1, "b200moe_ep_p2p_return", _p(rows), _p(dw_rows), _p(plan),
            _p(peer_rows), _p(peer_dw), n, H, k, ranks, _s(rows))


def ep_p2p_reduce_return(rows, d: Dispatch, plan, peer_rows, ranks: int, weights=None,
                         dw_rows=None, peer_dw=None):
    """Owner side: each received row's sum over its local slots (weighted: the
    combine; unweighted: the gather backward) stored into the source's back rows."""
    H = rows.shape[1]
    _launch("ep_p2p_reduce_return", 1, "b200moe_ep_p2p_reduce_return", _p(rows), _p(d.inv_pad),
            _p(weights), d.top_k, _p(dw_rows), _p(plan), _p(peer_rows), _p(peer_dw),
            d.num_tokens, H, ranks, _s(rows))


def ep_p2p_back_inv(send: Dispatch, plan) -> torch.Tensor:
    T, P = send.num_tokens, send.num_experts
    inv = torch.empty(max(T * P, 1), device=plan.device, dtype=torch.int32)
    if T == 0:
        return inv[:0]
    _launch("ep_p2p_back_inv", 1, "b200moe_ep_p2p_back_inv", _p(send.inv_pad),
            _p(send.pad_offsets), _p(plan), T, P, _p(inv), _s(plan))
    return inv[: T * P]


def ep_barrier(peer_flags, my_flags, me: int, ranks: int, epoch: int):
    _launch("ep_barrier", 1, "b200moe_ep_barrier", _p(peer_flags), _p(my_flags), me, ranks,
            ctypes.c_ulonglong(epoch), _s(my_flags))


def ep_weight_grad(dw_rows, send: Dispatch, selected, experts_per_rank: int,
                   out=None) -> torch.Tensor:
    T, k = selected.shape
    d_w = torch.empty(T, k, device=selected.device, dtype=torch.float32) if out is None else out
    if T:
        _launch("ep_weight_grad", 1, "b200moe_ep_weight_grad", _p(dw_rows), _p(send.inv_pad),
                _p(selected), T, k, experts_per_rank, send.num_experts, _p(d_w), _s(selected))
    return d_w


# --------------------------------------------------------------------------- #
# load-balancing loss (train.py:3098-3197)
# --------------------------------------------------------------------------- #
def lb_stats(logits, selected, valid_u8, num_experts, top_k, packed):
    T = logits.shape[0]
    nbytes = int(_lib.value("b200moe_lb_scratch_bytes", T, num_experts))
    scratch = torch.empty(nbytes, device=logits.device, dtype=torch.uint8)
    if T:
        _launch("lb_stats", 3, "b200moe_lb_stats", _p(logits), logits.stride(0), _p(selected),
                _p(valid_u8), T, num_experts, top_k, _p(packed), _p(scratch), nbytes,
                _s(logits))
    return packed


def lb_finalize(packed, num_experts, top_k, world):
    dev = packed.device
    aux = torch.empty((), device=dev, dtype=torch.float32)
    stats = torch.empty(5, device=dev, dtype=torch.float32)
    coef = torch.empty(num_experts, device=dev, dtype=torch.float32)
    _launch("lb_finalize", 1, "b200moe_lb_finalize", _p(packed), num_experts, top_k, world,
            _p(aux), _p(stats), _p(coef), _s(packed))
    return aux, stats, coef


def lb_grad(logits, valid_u8, coef, grad, num_experts):
    T, ld = logits.shape[0], logits.stride(0)
    out = torch.empty(T, ld, device=logits.device, dtype=BF16)
    if T:
        _launch("lb_grad", 1, "b200moe_lb_grad", _p(logits), ld, _p(valid_u8), T, num_experts,
                _p(coef), _p(grad), _p(out), _s(logits))
    return out


# --------------------------------------------------------------------------- #
# the training step around the layer: rows in bf16 or fp32, any row stride
# --------------------------------------------------------------------------- #
def as_rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """(..., cols) -> (rows, cols) with unit column stride, without a copy where
    the strides allow one."""
    if not t.is_cuda:
        raise RuntimeError(f"{name}: the B200 MoE kernels need CUDA tensors (no CPU path)")
    if t.dtype not in (BF16, torch.float32):
        raise RuntimeError(f"{name}: expected bf16 or fp32, got {t.dtype}")
    if t.dim() == 0 or not 0 < t.shape[-1] < 2 ** 31:
        raise RuntimeError(f"{name}: expected rows of one column or more and fewer than 2^31 columns, "
                           f"got shape {tuple(t.shape)}")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """Rows (as_rows) that could be read 16 bytes at a time but start elsewhere, copied to
    where they can be: a result then has the same bits wherever its input lies."""
    size = t.element_size()
    if t.shape[1] * size % 16 == 0 and (t.data_ptr() % 16 or t.stride(0) * size % 16):
        return t.clone(memory_format=torch.contiguous_format)
    return t


# In a traced model the training-step operators run between its graphs: their calls take pointers
# and streams, which a trace cannot hold.
outside_graph = torch.compiler.disable

_ENTRIES: dict = {}


def _entry(name: str):
    fn = _ENTRIES[name] = getattr(_lib.load(), name)
    return fn


def _call_on(t: torch.Tensor, label: str, kernels: int, name: str, *args) -> None:
    """Call entry point `name` with `args` and the current stream of t's device, which is
    made the current device if it is not (the library launches there).

    The short way: these operators are called on a few rows at a time, where the host's work is
    most of a call.  Pointers are plain integers (0 or None: null)."""
    dev = t.get_device()
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _call_on(t, label, kernels, name, *args)
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if _timing is not None and label in _timing:
        return _launch(label, kernels, name, *args, stream)
    LAUNCHES["count"] += kernels
    fn = _ENTRIES.get(name) or _entry(name)
    if fn(*args, stream) != 0:
        msg = _lib.load().b200moe_last_error().decode(errors="replace")
        raise RuntimeError(f"{name} failed: {msg}")


def _ptr(t):
    return None if t is None else t.data_ptr()


_CONTIGUOUS = torch.contiguous_format


def layer_norm_fwd(x, w, b, eps, save: bool, like=None):
    """x: rows (as_rows); w, b: (H,) contiguous fp32 or None.  -> y (contiguous, of the shape of
    `like` or x), stats ((2, T) fp32: mean and 1 / deviation of each row; None unless `save`)."""
    T, H = x.shape
    y = torch.empty_like(x if like is None else like, memory_format=_CONTIGUOUS)
    stats = mean = rstd = None
    if save:
        stats = x.new_empty((2, T), dtype=torch.float32)
        mean = stats.data_ptr()
        rstd = mean + 4 * T
    _call_on(x, "layer_norm", 1, "b200moe_layer_norm_fwd", x.data_ptr(),
             x.dtype is torch.float32, x.stride(0), _ptr(w), _ptr(b), T, H, eps, y.data_ptr(),
             mean, rstd)
    return y, stats


@lru_cache(maxsize=256)
def _norm_scratch_bytes(T: int, H: int, device: int) -> int:
    with torch.cuda.device(device):
        return _entry_value("b200moe_layer_norm_bwd_scratch_bytes", T, H)


def layer_norm_bwd(dy, x, w, stats, want_dx: bool, want_dw: bool, like=None):
    """-> dx (contiguous, of the shape of `like` or x), dw, db (None where not wanted); dy:
    rows of x's type; stats: the forward's."""
    T, H = x.shape
    dx = dw = db = scratch = None
    nbytes = 0
    if want_dx:
        dx = torch.empty_like(x if like is None else like, memory_format=_CONTIGUOUS)
    if want_dw:
        dw = x.new_empty(H, dtype=torch.float32) if w is None else torch.empty_like(w)
        db = torch.empty_like(dw)
        nbytes = _norm_scratch_bytes(T, H, x.get_device())
        scratch = x.new_empty(nbytes, dtype=torch.uint8)
    mean = stats.data_ptr()
    _call_on(x, "layer_norm_bwd", 1 + int(want_dw), "b200moe_layer_norm_bwd", dy.data_ptr(),
             dy.stride(0), x.data_ptr(), x.dtype is torch.float32, x.stride(0), _ptr(w), mean,
             mean + 4 * T, T, H, _ptr(dx), _ptr(dw), _ptr(db), _ptr(scratch), nbytes)
    return dx, dw, db


def _entry_value(name: str, *args) -> int:
    return (_ENTRIES.get(name) or _entry(name))(*args)


def route_experts_fwd(logits, bias, top_k, sigmoid, groups, kept, top2, normalize, scale):
    """logits: rows (as_rows).  -> weights (T, k) fp32, selected (T, k) int64."""
    T, E = logits.shape
    sel = logits.new_empty((T, top_k), dtype=torch.int64)
    w = logits.new_empty((T, top_k), dtype=torch.float32)
    _call_on(logits, "route_experts", 1, "b200moe_route_experts_fwd", logits.data_ptr(),
             logits.dtype is torch.float32, logits.stride(0), T, E, top_k, _ptr(bias), sigmoid,
             groups, kept, top2, normalize, scale, sel.data_ptr(), w.data_ptr())
    return w, sel


def records(*tensors) -> bool:
    """Whether a call goes through its autograd function: where a gradient is recorded, and inside
    a forward-mode level, where the function refuses a tangent (the kernels would drop it)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def refuse_second_order(name: str) -> None:
    """In a backward: grad mode is on there only with create_graph=True, whose graph would lack
    this operator's part."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name}: its gradient is not differentiable (create_graph=True)")


def route_experts_bwd(logits, selected, d_weights, sigmoid, normalize, scale):
    """-> d_logits (T, E) of the logits' type."""
    T, E = logits.shape
    out = torch.empty_like(logits, memory_format=_CONTIGUOUS)
    _call_on(logits, "route_experts_bwd", 1, "b200moe_route_experts_bwd", logits.data_ptr(),
             logits.dtype is torch.float32, logits.stride(0), selected.data_ptr(),
             d_weights.data_ptr(), T, E, selected.shape[1], sigmoid, normalize, scale,
             out.data_ptr())
    return out


def expert_counts(selected, num_experts: int) -> torch.Tensor:
    """(E,) int32 occurrences of each expert id (ids outside [0, E) are not counted)."""
    _check(selected, torch.int64, "expert_counts selected")
    out = selected.new_empty(num_experts, dtype=torch.int32)
    _call_on(selected, "expert_counts", 1, "b200moe_expert_counts", selected.data_ptr(),
             selected.numel(), num_experts, out.data_ptr())
    return out


def balance_bias(bias, counts, rate: float) -> torch.Tensor:
    """bias + rate * sign(mean(counts) - counts), counts (E,) int32."""
    _check(bias, torch.float32, "balance_bias bias")
    _check(counts, torch.int32, "balance_bias counts")
    out = torch.empty_like(bias)
    _call_on(bias, "balance_bias", 1, "b200moe_balance_bias", bias.data_ptr(), counts.data_ptr(),
             bias.numel(), rate, out.data_ptr())
    return out


def balance_step(bias, selected, rate: float) -> torch.Tensor:
    """balance_bias of the counts of `selected`, in one launch."""
    _check(bias, torch.float32, "balance_bias bias")
    _check(selected, torch.int64, "balance_bias selected")
    E = bias.numel()
    out = torch.empty_like(bias)
    scratch = selected.new_empty(E + 1, dtype=torch.int32)
    _call_on(bias, "balance_step", 1, "b200moe_balance_step", selected.data_ptr(),
             selected.numel(), E, bias.data_ptr(), rate, scratch.data_ptr(), out.data_ptr())
    return out


def token_logprobs_fwd(logits, tokens, top, temperature, ignore, save: bool):
    """logits: rows (as_rows); tokens (T,) int64 contiguous.  -> logprob, entropy,
    top_logprobs, top_ids (None, None for top = 0), stats (None unless `save`)."""
    T, V = logits.shape
    logprob = logits.new_empty(T, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    top_lp = top_ids = stats = None
    if top:
        top_lp = logits.new_empty((T, top), dtype=torch.float32)
        top_ids = logits.new_empty((T, top), dtype=torch.int64)
    if save:
        stats = logits.new_empty((T, 2), dtype=torch.float32)
    _call_on(logits, "token_logprobs", 1, "b200moe_token_logprobs_fwd", logits.data_ptr(),
             logits.dtype is torch.float32, logits.stride(0), tokens.data_ptr(), T, V,
             temperature, ignore, top, logprob.data_ptr(), entropy.data_ptr(), _ptr(top_lp),
             _ptr(top_ids), _ptr(stats))
    return logprob, entropy, top_lp, top_ids, stats


def token_logprobs_bwd(logits, tokens, stats, entropy, d_logprob, d_entropy, temperature, ignore):
    """-> d_logits (T, V) of the logits' type; d_logprob, d_entropy (T,) fp32 or None.

    Its rows lie in memory as the logits' do, with the padding of a vocabulary cut to V and the
    offset from a 16-byte boundary, so that the kernel moves whole vectors (4096 x 50257 bf16
    cut from 50304: 197 us into a contiguous gradient, 130 so); with more than an eighth of
    padding they are contiguous."""
    T, V = logits.shape
    ld, off = logits.stride(0), logits.data_ptr() % 16 // logits.element_size()
    if ld == V and not off:
        out = torch.empty_like(logits, memory_format=_CONTIGUOUS)
    else:
        if not V <= ld <= V + V // 8:
            ld = V
        out = logits.new_empty(off + T * ld).as_strided((T, V), (ld, 1), off)
    _call_on(logits, "token_logprobs_bwd", 1, "b200moe_token_logprobs_bwd", logits.data_ptr(),
             logits.dtype is torch.float32, logits.stride(0), tokens.data_ptr(), T, V,
             temperature, ignore, stats.data_ptr(), entropy.data_ptr(), _ptr(d_logprob),
             _ptr(d_entropy), out.data_ptr(), ld)
    return out


_GRAD_KINDS = {torch.float32: 1, BF16: 0}


class GradList:
    """Host arrays (pointers, element counts, types) of a list of gradients, as the
    library's gradient entry points take them."""

    def __init__(self, tensors, name: str):
        self.tensors = tensors
        devices = set(map(torch.Tensor.get_device, tensors))
        if len(devices) > 1 or -1 in devices:
            raise RuntimeError(f"{name}: the gradients must be CUDA tensors of one device")
        try:
            self.kinds = array("i", [_GRAD_KINDS[t.dtype] for t in tensors])
        except KeyError as e:
            raise RuntimeError(f"{name}: expected bf16 or fp32 gradients, got {e.args[0]}") from None
        if not all(map(torch.Tensor.is_contiguous, tensors)):
            raise RuntimeError(f"{name}: the gradients must be contiguous")
        if forward_ad._current_level >= 0 and any(
                forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise RuntimeError(f"{name}: it has no forward-mode derivative")
        self.ptrs = array("q", list(map(torch.Tensor.data_ptr, tensors)))
        self.sizes = array("q", list(map(torch.Tensor.numel, tensors)))

    def written(self) -> None:
        """Tell autograd that the tensors were changed in place."""
        torch.autograd.graph.increment_version(self.tensors)

    def args(self):
        return self.ptrs.buffer_info()[0], self.sizes.buffer_info()[0], self.kinds.buffer_info()[0]


@lru_cache(maxsize=1)
def _grad_partials_count() -> int:
    return _entry_value("b200moe_grad_partials_count")


def _grad_partials_buffer(like: torch.Tensor) -> torch.Tensor:
    return like.new_empty(_grad_partials_count(), dtype=torch.float64)


def grad_partials(grads: GradList, inf_norm: bool) -> torch.Tensor:
    """fp64 partial sums of squares (or maxima) of the gradients, a fixed number of them."""
    first = grads.tensors[0]
    out = _grad_partials_buffer(first)
    ptrs, sizes, kinds = grads.args()
    _call_on(first, "grad_norm", 1, "b200moe_grad_partials", ptrs, sizes, kinds,
             len(grads.tensors), inf_norm, out.data_ptr())
    return out


def grad_clip(grads: GradList | None, inf_norm: bool, partials, max_norm: float) -> torch.Tensor:
    """Scale the gradients in place by the norm that the partials give, which is returned
    (0-d fp32).  grads None: the norm alone."""
    norm = partials.new_empty((), dtype=torch.float32)
    ptrs = sizes = kinds = None
    n = 0
    if grads is not None:
        ptrs, sizes, kinds = grads.args()
        n = len(grads.tensors)
    _call_on(partials, "grad_clip", 1, "b200moe_grad_clip", ptrs, ptrs, sizes, kinds, n, inf_norm,
             partials.data_ptr(), partials.numel(), max_norm, norm.data_ptr())
    if grads is not None:
        grads.written()
    return norm


def clip_grads(grads: GradList, out: GradList, inf_norm: bool, max_norm: float) -> torch.Tensor:
    """grad_partials and the scaling into `out` in one call; returns the norm (0-d fp32)."""
    first = grads.tensors[0]
    partials = _grad_partials_buffer(first)
    norm = first.new_empty((), dtype=torch.float32)
    ptrs, sizes, kinds = grads.args()
    _call_on(first, "clip_grads", 2, "b200moe_clip_grads", ptrs, out.ptrs.buffer_info()[0], sizes,
             kinds, len(grads.tensors), inf_norm, partials.data_ptr(), max_norm, norm.data_ptr())
    out.written()
    return norm
