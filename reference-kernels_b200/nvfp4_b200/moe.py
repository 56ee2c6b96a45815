"""Mixture of experts on the GPU: tokens sorted by expert and back, with weights
applied, their gradients, and the experts' MLP with MXFP4 weights.

Each of T tokens has ``top`` slots, each with the number of an expert.
``sort`` gives every slot a row, by expert; numbers outside 0 .. experts-1 are
not routed (experts of another rank: subtract this rank's first; dropped slots:
-1).  The routing stays on the GPU: buffers of sorted rows have T*top rows
however many are routed, and rows behind the last expert's are zeros in every
value that a function here returns.

    routing = moe.sort(ids, experts)
    xs = moe.gather(x, routing)                    # [T*top, H]
    ys = ...                                       # the experts, on rows sorted by expert
    y = moe.combine(ys, weights, routing)          # [T, H]

    dys, dweights = moe.combine_backward(dy, ys, weights, routing)
    dx = moe.gather_backward(dxs, routing)

Sums are in fp32, in the order of the slots, so that results are the same on
every run.  Launches go to the current CUDA stream; nothing is synchronised, and
everything can be captured into a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, mx
from .inputs import FP4X2
from .mx import _DTYPES, _byref, _device, _experts, _raw_stream, _require, E8M0, scale_blocks


class Routing(NamedTuple):
    """order int32 [T*top]: the slot (token * top + choice) of each sorted row, -1 behind the last;
    slots int32 [T, top]: the sorted row of each slot, -1 where it is not routed;
    offsets int32 [experts + 1]: each expert's first row, and the number of rows."""
    order: torch.Tensor
    slots: torch.Tensor
    offsets: torch.Tensor


def sort(ids: torch.Tensor, experts: int) -> Routing:
    """Sorts the slots of ids [T, top] (int32 or int64, contiguous) by expert, stably; at most 1024 experts."""
    who = "moe.sort"
    _require(ids.dtype in (torch.int32, torch.int64), f"{who}: ids must be int32 or int64, got {ids.dtype}")
    _require(ids.dim() == 2 and ids.is_contiguous(), f"{who}: ids must be contiguous [tokens, top], "
             f"got {tuple(ids.shape)} (strides {ids.stride()})")
    dev = _device(who, ids)
    n = ids.numel()
    lib = _lib.load()
    need = lib.nvfp4_moe_sort_workspace(n, experts)
    _require(need >= 0, f"{who}: experts={experts} must be 1 to 1024")
    order = torch.empty((n,), dtype=torch.int32, device=ids.device)
    slots = torch.empty(ids.shape, dtype=torch.int32, device=ids.device)
    offsets = torch.empty((experts + 1,), dtype=torch.int32, device=ids.device)
    # On the caching allocator: a call on another stream, or a captured one, has its own.
    work = torch.empty((need,), dtype=torch.uint8, device=ids.device) if need else None
    _lib.check(lib.nvfp4_moe_sort(ids.data_ptr(), ids.element_size(), n, experts, order.data_ptr(), slots.data_ptr(),
                                  offsets.data_ptr(), work.data_ptr() if need else None, need, _raw_stream(dev)))
    return Routing(order, slots, offsets)


def _check_routing(who: str, routing: Routing):
    """(tokens, top, experts) of a routing."""
    order, slots, offsets = routing
    _require(slots.dtype == torch.int32 and slots.dim() == 2 and slots.is_contiguous(),
             f"{who}: routing.slots must be contiguous int32 [tokens, top]")
    return slots.shape[0], slots.shape[1], _experts(who, offsets)


def _check_matrix(who: str, name: str, t: torch.Tensor, rows: int, like: torch.Tensor | None = None) -> None:
    _require(t.dtype in _DTYPES, f"{who}: {name} must be fp16, bf16 or fp32, got {t.dtype}")
    _require(t.dim() == 2 and t.shape[0] == rows, f"{who}: {name} must be [{rows}, hidden], got {tuple(t.shape)}")
    _require(t.stride(1) == 1 or t.shape[1] <= 1, f"{who}: {name} must have unit stride along the hidden dimension "
             f"(strides {t.stride()})")
    _require(like is None or (t.dtype == like.dtype and t.shape[1] == like.shape[1]),
             f"{who}: {name} must have the other operand's type and hidden size")


def _check_weights(who: str, weights: torch.Tensor, routing: Routing) -> None:
    _require(weights.dtype == torch.float32 and weights.shape == routing.slots.shape and weights.is_contiguous(),
             f"{who}: weights must be contiguous fp32 {tuple(routing.slots.shape)}, "
             f"got {weights.dtype} {tuple(weights.shape)} (strides {weights.stride()})")


def gather(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """x [T, H] -> xs [T*top, H], each token's row at each of its sorted rows."""
    who = "moe.gather"
    tokens, top, experts = _check_routing(who, routing)
    _check_matrix(who, "x", x, tokens)
    dev = _device(who, x, routing.slots, routing.offsets)
    h = x.shape[1]
    xs = torch.empty((tokens * top, h), dtype=x.dtype, device=x.device)
    _lib.check(_lib.load().nvfp4_moe_gather(_byref(_lib.MoeArgs(
        x.data_ptr(), None, None, xs.data_ptr(), None, routing.slots.data_ptr(), routing.offsets.data_ptr(),
        _DTYPES[x.dtype], tokens, top, h, experts, 0, x.stride(0), 0, _raw_stream(dev)))))
    return xs


def gather_backward(dxs: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The gradient of gather: dxs [T*top, H] -> dx [T, H], the sum over each token's rows."""
    who = "moe.gather_backward"
    tokens, top, experts = _check_routing(who, routing)
    _check_matrix(who, "dxs", dxs, tokens * top)
    dev = _device(who, dxs, routing.slots)
    h = dxs.shape[1]
    dx = torch.empty((tokens, h), dtype=dxs.dtype, device=dxs.device)
    _lib.check(_lib.load().nvfp4_moe_gather_backward(_byref(_lib.MoeArgs(
        dxs.data_ptr(), None, None, dx.data_ptr(), None, routing.slots.data_ptr(), None,
        _DTYPES[dxs.dtype], tokens, top, h, experts, 0, dxs.stride(0), 0, _raw_stream(dev)))))
    return dx


def combine(ys: torch.Tensor, weights: torch.Tensor, routing: Routing) -> torch.Tensor:
    """ys [T*top, H], weights fp32 [T, top] -> y [T, H], the weighted sum of each token's rows (no row: zeros)."""
    who = "moe.combine"
    tokens, top, experts = _check_routing(who, routing)
    _check_matrix(who, "ys", ys, tokens * top)
    _check_weights(who, weights, routing)
    dev = _device(who, ys, weights, routing.slots)
    h = ys.shape[1]
    y = torch.empty((tokens, h), dtype=ys.dtype, device=ys.device)
    _lib.check(_lib.load().nvfp4_moe_combine(_byref(_lib.MoeArgs(
        ys.data_ptr(), None, weights.data_ptr(), y.data_ptr(), None, routing.slots.data_ptr(), None,
        _DTYPES[ys.dtype], tokens, top, h, experts, 0, ys.stride(0), 0, _raw_stream(dev)))))
    return y


def combine_backward(dy: torch.Tensor, ys: torch.Tensor, weights: torch.Tensor, routing: Routing):
    """The gradients of combine: (dys [T*top, H], dweights fp32 [T, top])."""
    who = "moe.combine_backward"
    tokens, top, experts = _check_routing(who, routing)
    _check_matrix(who, "dy", dy, tokens)
    _check_matrix(who, "ys", ys, tokens * top, dy)
    _check_weights(who, weights, routing)
    dev = _device(who, dy, ys, weights, routing.slots, routing.offsets)
    h = dy.shape[1]
    dys = torch.empty((tokens * top, h), dtype=ys.dtype, device=ys.device)
    dweights = torch.empty((tokens, top), dtype=torch.float32, device=ys.device)
    _lib.check(_lib.load().nvfp4_moe_combine_backward(_byref(_lib.MoeArgs(
        ys.data_ptr(), dy.data_ptr(), weights.data_ptr(), dys.data_ptr(), dweights.data_ptr(),
        routing.slots.data_ptr(), routing.offsets.data_ptr(), _DTYPES[ys.dtype], tokens, top, h, experts, 0,
        ys.stride(0), dy.stride(0), _raw_stream(dev)))))
    return dys, dweights


def quantize_tokens(x: torch.Tensor, routing: Routing):
    """x [T, H] (fp16, bf16 or fp32, H % 32 == 0) -> the MXFP4 operand (packed [T*top, H/2], scales) of its sorted
    rows: mx.quantize of gather(x), with each token quantised once.  Rows behind the last expert's are not written."""
    who = "moe.quantize_tokens"
    tokens, top, experts = _check_routing(who, routing)
    _check_matrix(who, "x", x, tokens)
    h = x.shape[1]
    _require(h > 0 and h % 32 == 0, f"{who}: hidden={h} must be a positive multiple of 32")
    dev = _device(who, x, routing.slots, routing.offsets)
    rows = tokens * top
    packed = torch.empty((rows, h // 2), dtype=FP4X2, device=x.device)
    scales = torch.empty((scale_blocks(rows, experts), -(-h // 128), 32, 4, 4), dtype=E8M0, device=x.device)
    if rows:
        _lib.check(_lib.load().nvfp4_mx_quantize(_byref(_lib.MxQuantArgs(
            x.data_ptr(), packed.data_ptr(), scales.data_ptr(), routing.offsets.data_ptr(), routing.slots.data_ptr(),
            _DTYPES[x.dtype], tokens, h, experts, top, 0, x.stride(0), 0, _raw_stream(dev)))))
    return packed, scales


def mlp(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, gate, up, down) -> torch.Tensor:
    """The experts' MLP on x [T, H]: y[t] = sum_j weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])), e = ids[t, j].

    gate, up: operands (packed, scales) of [experts, N, H] weights, down of [experts, H, N], as mx.quantize makes them
    (H and N multiples of 32); ids [T, top] as for sort, weights fp32 [T, top].  The tokens and the gated values are
    quantised to MXFP4 on the way; x and the result are fp16, bf16 or fp32, and so are the values between the
    products.  Six launches (seven for more than 4096 slots), no synchronisation."""
    _require(gate[0].dim() == 3, f"moe.mlp: gate must be weights [experts, N, H/2], got {tuple(gate[0].shape)}")
    routing = sort(ids, gate[0].shape[0])
    h = mx.dual_gemm(*quantize_tokens(x, routing), *gate, *up, offsets=routing.offsets, out_dtype=x.dtype)
    y = mx.gemm(*mx.quantize(h, offsets=routing.offsets), *down, offsets=routing.offsets, out_dtype=x.dtype)
    return combine(y, weights, routing)
