"""Mixture of experts on the GPU: tokens sorted by expert and back, with weights
applied, their gradients, and the experts' MLP with MXFP4 weights.

Each of T tokens has ``top`` slots, each with the number of an expert.
``sort`` gives every slot a row, by expert; numbers outside 0 .. experts-1 are
not routed (experts of another rank: subtract this rank's first; dropped slots:
-1).  The routing stays on the GPU: buffers of sorted rows have T*top rows
however many are routed, and rows that no expert has (behind the last one's, or
in front of the first one's where a Routing has the offsets of some of the
experts only) are zeros in every value that a function here returns.

    routing = moe.sort(ids, experts)
    xs = moe.gather(x, routing)                    # [T*top, H]
    ys = ...                                       # the experts, on rows sorted by expert
    y = moe.combine(ys, weights, routing)          # [T, H]

    dys, dweights = moe.combine_backward(dy, ys, weights, routing)
    dx = moe.gather_backward(dxs, routing)

Gradients are these functions; nothing here records a graph for autograd, and
gather, combine and mlp refuse inputs that require grad while grad mode is on,
where a result without a graph would lose the gradient.  Call them under
torch.no_grad(), as the forward of a torch.autograd.Function is.

Sums are in fp32, in the order of the slots, so that results are the same on
every run.  Launches go to the current CUDA stream; nothing is synchronised, and
everything can be captured into a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, mx
from .inputs import FP4X2
from .mx import _DTYPES, _device, _experts, _fail, _launch, _raw_stream, E8M0, scale_blocks


class _Lists(NamedTuple):
    order: torch.Tensor
    slots: torch.Tensor
    offsets: torch.Tensor


class Routing(_Lists):
    """order int32 [T*top]: the slot (token * top + choice) of each sorted row, -1 behind the last;
    slots int32 [T, top]: the sorted row of each slot, -1 where it is not routed;
    offsets int32 [experts + 1]: each expert's first row, from 0 on, and the number of rows; or the part of them for
    some of the experts in turn, whose rows alone then count: a slot with a row outside them is as one not routed.

    One made by hand gives each row of those experts to one slot: with a row in two slots the two tokens' values mix in
    it, and a row in none is not written.
    slots and offsets are checked once, when it is made (order is for the caller: nothing here reads it); tokens,
    top, experts and device (its CUDA index) are plain attributes."""

    def __new__(cls, order, slots, offsets):
        shape = slots.shape
        if len(shape) != 2 or slots.dtype is not torch.int32 or not slots.is_contiguous():
            _fail("moe.Routing: slots must be contiguous int32 [tokens, top]")
        self = tuple.__new__(cls, (order, slots, offsets))
        self.tokens, self.top = shape
        self.experts = _experts("moe.Routing", offsets)
        self.device = slots.get_device()
        if offsets.get_device() != self.device:
            _fail("moe.Routing: slots and offsets must be on one device")
        return self

    @classmethod
    def _make(cls, lists):
        return cls(*lists)


def sort(ids: torch.Tensor, experts: int) -> Routing:
    """Sorts the slots of ids [T, top] (int32 or int64, contiguous) by expert, stably; at most 1024 experts."""
    who = "moe.sort"
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        _fail(f"{who}: ids must be int32 or int64, got {ids.dtype}")
    shape = ids.shape
    if len(shape) != 2 or not ids.is_contiguous():
        _fail(f"{who}: ids must be contiguous [tokens, top], got {tuple(shape)} (strides {ids.stride()})")
    dev = _device(who, ids)
    n = shape[0] * shape[1]
    if n >= (1 << 31) - (1 << 20):
        _fail(f"{who}: {n} slots do not fit 32-bit rows")
    if not 1 <= experts <= 1024:
        _fail(f"{who}: experts={experts} must be 1 to 1024")
    lib = _lib.load()
    need = lib.nvfp4_moe_sort_workspace(n, experts)
    order = ids.new_empty((n,), dtype=torch.int32)
    slots = ids.new_empty(shape, dtype=torch.int32)
    offsets = ids.new_empty((experts + 1,), dtype=torch.int32)
    # On the caching allocator: a call on another stream, or a captured one, has its own.
    work = ids.new_empty((need,), dtype=torch.uint8) if need else None
    rc = lib.nvfp4_moe_sort(ids.data_ptr(), ids.element_size(), n, experts, order.data_ptr(), slots.data_ptr(),
                            offsets.data_ptr(), work.data_ptr() if need else None, need, _raw_stream(dev))
    if rc:
        _lib.check(rc)
    routing = tuple.__new__(Routing, (order, slots, offsets))  # nothing to check
    routing.tokens, routing.top = shape
    routing.experts, routing.device = experts, dev
    return routing


def _on(who: str, routing: Routing, t: torch.Tensor, *others) -> int:
    """The device of the routing and of every tensor, which has to be the current one."""
    dev = _device(who, t, *others)
    if routing.device != dev:
        _fail(f"{who}: the routing is on cuda:{routing.device}, {who.split('.')[1]}'s tensors on cuda:{dev}")
    return dev


def _no_graph(who: str) -> None:
    """For inputs of which one requires grad."""
    if torch.is_grad_enabled():
        _fail(f"{who}: an input requires grad, but no graph is recorded; call under torch.no_grad() "
              f"(moe.gather_backward and moe.combine_backward are the gradients)")


def _check_matrix(who: str, name: str, t: torch.Tensor, rows: int):
    """(dtype code, hidden, row stride) of t [rows, hidden]."""
    code = _DTYPES.get(t.dtype)
    if code is None:
        _fail(f"{who}: {name} must be fp16, bf16 or fp32, got {t.dtype}")
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows:
        _fail(f"{who}: {name} must be [{rows}, hidden], got {tuple(shape)}")
    stride, unit = t.stride()
    if unit != 1 and shape[1] > 1:
        _fail(f"{who}: {name} must have unit stride along the hidden dimension (strides {t.stride()})")
    return code, shape[1], stride


def _check_weights(who: str, weights: torch.Tensor, routing: Routing) -> None:
    want = (routing.tokens, routing.top)
    if weights.dtype is not torch.float32 or weights.shape != want or not weights.is_contiguous():
        _fail(f"{who}: weights must be contiguous fp32 {want}, "
              f"got {weights.dtype} {tuple(weights.shape)} (strides {weights.stride()})")


def _rows(name, routing, x, grad, weights, out, dweights, code, h, stride, gstride, dev):
    """One of the nvfp4_moe_* entry points that take nvfp4_moe_args."""
    _, slots, offsets = routing
    rc = getattr(_lib.load(), name)(_lib.pack_moe(
        x.data_ptr(), 0 if grad is None else grad.data_ptr(), 0 if weights is None else weights.data_ptr(),
        out.data_ptr(), 0 if dweights is None else dweights.data_ptr(), slots.data_ptr(), offsets.data_ptr(), code,
        routing.tokens, routing.top, h, routing.experts, 0, stride, gstride, _raw_stream(dev)))
    if rc:
        _lib.check(rc)


def gather(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """x [T, H] -> xs [T*top, H], each token's row at each of its sorted rows."""
    who = "moe.gather"
    tokens = routing.tokens
    code, h, stride = _check_matrix(who, "x", x, tokens)
    if x.requires_grad:
        _no_graph(who)
    dev = _on(who, routing, x)
    xs = x.new_empty((tokens * routing.top, h))
    _rows("nvfp4_moe_gather", routing, x, None, None, xs, None, code, h, stride, 0, dev)
    return xs


def gather_backward(dxs: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The gradient of gather: dxs [T*top, H] -> dx [T, H], the sum over each token's rows."""
    who = "moe.gather_backward"
    tokens = routing.tokens
    code, h, stride = _check_matrix(who, "dxs", dxs, tokens * routing.top)
    dev = _on(who, routing, dxs)
    dx = dxs.new_empty((tokens, h))
    _rows("nvfp4_moe_gather_backward", routing, dxs, None, None, dx, None, code, h, stride, 0, dev)
    return dx


def combine(ys: torch.Tensor, weights: torch.Tensor, routing: Routing) -> torch.Tensor:
    """ys [T*top, H], weights fp32 [T, top] -> y [T, H], the weighted sum of each token's rows (no row: zeros)."""
    who = "moe.combine"
    tokens = routing.tokens
    code, h, stride = _check_matrix(who, "ys", ys, tokens * routing.top)
    _check_weights(who, weights, routing)
    if ys.requires_grad or weights.requires_grad:
        _no_graph(who)
    dev = _on(who, routing, ys, weights)
    y = ys.new_empty((tokens, h))
    _rows("nvfp4_moe_combine", routing, ys, None, weights, y, None, code, h, stride, 0, dev)
    return y


def combine_backward(dy: torch.Tensor, ys: torch.Tensor, weights: torch.Tensor, routing: Routing):
    """The gradients of combine: (dys [T*top, H], dweights fp32 [T, top])."""
    who = "moe.combine_backward"
    tokens, rows = routing.tokens, routing.tokens * routing.top
    code, h, gstride = _check_matrix(who, "dy", dy, tokens)
    ycode, yh, stride = _check_matrix(who, "ys", ys, rows)
    if ycode != code or yh != h:
        _fail(f"{who}: ys must have dy's type and hidden size")
    _check_weights(who, weights, routing)
    dev = _on(who, routing, dy, ys, weights)
    dys = ys.new_empty((rows, h))
    dweights = weights.new_empty((tokens, routing.top))
    _rows("nvfp4_moe_combine_backward", routing, ys, dy, weights, dys, dweights, code, h, stride, gstride, dev)
    return dys, dweights


def quantize_tokens(x: torch.Tensor, routing: Routing):
    """x [T, H] (fp16, bf16 or fp32, H % 32 == 0) -> the MXFP4 operand (packed [T*top, H/2], scales) of its sorted
    rows: mx.quantize of gather(x), with each token quantised once.  Rows that no expert has are not written."""
    who = "moe.quantize_tokens"
    _, slots, offsets = routing
    tokens, top, experts = routing.tokens, routing.top, routing.experts
    code, h, stride = _check_matrix(who, "x", x, tokens)
    if h == 0 or h % 32:
        _fail(f"{who}: hidden={h} must be a positive multiple of 32")
    dev = _on(who, routing, x)
    rows = tokens * top
    packed = x.new_empty((rows, h // 2), dtype=FP4X2)
    scales = x.new_empty((scale_blocks(rows, experts), -(-h // 128), 32, 4, 4), dtype=E8M0)
    if rows:
        _launch("nvfp4_mx_quantize", x, packed, scales, offsets, slots, code, tokens, h, experts, top, 0, stride, 0,
                dev)
    return packed, scales


def mlp(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, gate, up, down) -> torch.Tensor:
    """The experts' MLP on x [T, H]: y[t] = sum_j weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])),
    e = ids[t, j].

    gate, up: operands (packed, scales) of [experts, N, H] weights, down of [experts, H, N], as mx.quantize makes them
    (H and N multiples of 32); ids [T, top] as for sort, weights fp32 [T, top].  x and the result are fp16, bf16 or
    fp32; the tokens are quantised to MXFP4 as they are sorted, the gated values in the product's epilogue, and the
    down projection's rows have x's type.  Five launches (six for more than 32768 slots), no synchronisation."""
    if x.requires_grad or weights.requires_grad:
        _no_graph("moe.mlp")
    if gate[0].dim() != 3:
        _fail(f"moe.mlp: gate must be weights [experts, N, H/2], got {tuple(gate[0].shape)}")
    routing = sort(ids, gate[0].shape[0])
    offsets = routing.offsets
    h = mx.dual_gemm(*quantize_tokens(x, routing), *gate, *up, offsets=offsets, quantize=True)
    return combine(mx.gemm(*h, *down, offsets=offsets, out_dtype=x.dtype), weights, routing)
