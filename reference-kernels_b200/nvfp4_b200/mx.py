"""MXFP4 (OCP microscaling: e2m1 values, one e8m0 scale per 32) on the GPU:
quantise, dequantise, and the products of quantised operands.

An operand is a pair ``(packed, scales)``:

* ``packed``: float4_e2m1fn_x2 ``[rows, K/2]`` (or ``[E, rows, K/2]``: E
  matrices), contiguous, the even K index in the low nibble;
* ``scales``: float8_e8m0fnu ``[ceil(rows/128), ceil(K/128), 32, 4, 4]`` (with a
  leading E), contiguous: the 128x4-blocked order in which the tensor cores
  read them.  Row ``r`` and block ``j`` of 32 are at ``[r//128, j//4, r%32,
  (r%128)//32, j%4]``; padding rows and columns hold anything.

uint8 tensors of the same shapes are taken as well.

Rows sorted by expert (``offsets``, int32 ``[experts + 1]`` on the GPU, as
``moe.sort`` returns): ``packed`` holds all rows without gaps, ``scales`` has
``min(rows, experts) + rows//128`` row blocks, and each expert's rows begin a
new one.  Nothing here reads the offsets on the host.

Launches go to the current CUDA stream; nothing is synchronised, and everything
can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .inputs import FP4X2
from .ops import _post

E8M0 = torch.float8_e8m0fnu
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_byref = ctypes.byref


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise _lib.Nvfp4Error(msg)


def _device(who: str, t: torch.Tensor, *others) -> int:
    """The device of every tensor (None: not given), which has to be the current one."""
    dev = t.get_device()
    _require(dev >= 0, f"{who}: expected a CUDA tensor (no CPU fallback)")
    for o in others:
        if o is not None and o.get_device() != dev:
            _require(False, f"{who}: tensors on different devices (cuda:{dev} and {o.device})")
    _require(dev == _current_device(),
             f"{who}: the tensors are on cuda:{dev} but cuda:{_current_device()} is current; "
             f"call inside torch.cuda.device({dev})")
    return dev


def _experts(who: str, offsets: torch.Tensor) -> int:
    _require(offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.is_contiguous()
             and 2 <= offsets.shape[0] <= 1025,
             f"{who}: offsets must be a contiguous int32 [experts + 1], at most 1024 experts")
    return offsets.shape[0] - 1


def scale_blocks(rows: int, experts: int | None = None) -> int:
    """Row blocks of the scales of ``rows`` rows (sorted by expert: for any offsets)."""
    return -(-rows // 128) if experts is None else min(rows, experts) + rows // 128


def _check_operand(who: str, packed: torch.Tensor, scales: torch.Tensor, dim: int, experts: int | None = None):
    """(matrices, rows, K) of an operand; ``dim``: of packed; ``experts``: rows are sorted by expert."""
    _require(packed.element_size() == 1 and packed.dim() == dim and packed.is_contiguous(),
             f"{who}: codes must be contiguous float4_e2m1fn_x2 or uint8 of {dim} dimensions, "
             f"got {packed.dtype} {tuple(packed.shape)} (strides {packed.stride()})")
    rows, k = packed.shape[-2], 2 * packed.shape[-1]
    _require(k > 0 and k % 32 == 0, f"{who}: K={k} must be a positive multiple of 32")
    want = (scale_blocks(rows, experts), -(-k // 128), 32, 4, 4)
    if dim == 3:
        want = (packed.shape[0], *want)
    _require(scales.element_size() == 1 and tuple(scales.shape) == want and scales.is_contiguous(),
             f"{who}: scales must be contiguous float8_e8m0fnu or uint8 {want}, "
             f"got {scales.dtype} {tuple(scales.shape)} (strides {scales.stride()})")
    return (packed.shape[0] if dim == 3 else 1), rows, k


def quantize(x: torch.Tensor, axis: int = -1, offsets: torch.Tensor | None = None):
    """x: [rows, K] or [E, rows, K] of fp16, bf16 or fp32 with unit stride along K -> (packed, scales).

    Per block of 32 along K (K % 32 == 0): the scale is 2^e, e =
    floor(log2(amax)) - 2 (at least -127), and the values x / 2^e rounded to
    e2m1, ties to even, magnitudes above 6 to 6.  A block that holds a NaN or an
    infinity becomes a NaN block.

    axis=0 (x [rows, K], any K): blocks run down the columns and the result is
    the quantised transpose, [K, rows] with rows padded with zeros to a multiple
    of 32: the operand of a product that sums over the rows, such as a weight
    gradient.

    offsets: the rows are sorted by expert.  Codes of rows behind the last
    expert's are not written."""
    who = "mx.quantize"
    _require(x.dtype in _DTYPES, f"{who}: x must be fp16, bf16 or fp32, got {x.dtype}")
    _require(x.dim() in (2, 3), f"{who}: x must be [rows, K] or [experts, rows, K], got {tuple(x.shape)}")
    rows, k = x.shape[-2:]
    columns = x.dim() == 2 and axis == 0
    _require(columns or axis in (-1, x.dim() - 1), f"{who}: axis={axis} must be the last, or 0 of a matrix")
    _require(k > 0 and (columns or k % 32 == 0), f"{who}: K={k} must be a positive multiple of 32")
    _require(x.stride(-1) == 1 or k == 1, f"{who}: x must have unit stride along K (strides {x.stride()})")
    dev = _device(who, x, offsets)
    experts = x.shape[0] if x.dim() == 3 else 1
    if columns:
        _require(offsets is None, f"{who}: axis=0 takes no offsets")
        kt = -(-rows // 32) * 32
        packed = torch.empty((k, kt // 2), dtype=FP4X2, device=x.device)
        scales = torch.empty((-(-k // 128), -(-kt // 128), 32, 4, 4), dtype=E8M0, device=x.device)
    elif offsets is not None:
        _require(x.dim() == 2, f"{who}: offsets need x [rows, K]")
        experts = _experts(who, offsets)
        packed = torch.empty((rows, k // 2), dtype=FP4X2, device=x.device)
        scales = torch.empty((scale_blocks(rows, experts), -(-k // 128), 32, 4, 4), dtype=E8M0, device=x.device)
    else:
        packed = torch.empty((*x.shape[:-1], k // 2), dtype=FP4X2, device=x.device)
        scales = torch.empty((*x.shape[:-2], -(-rows // 128), -(-k // 128), 32, 4, 4), dtype=E8M0, device=x.device)
    if packed.numel():
        args = _lib.MxQuantArgs(x.data_ptr(), packed.data_ptr(), scales.data_ptr(),
                                None if offsets is None else offsets.data_ptr(), None, _DTYPES[x.dtype], rows, k,
                                experts, 0, columns, x.stride(-2), x.stride(0) if x.dim() == 3 else 0,
                                _raw_stream(dev))
        _lib.check(_lib.load().nvfp4_mx_quantize(_byref(args)))
    return packed, scales


def dequantize(packed: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an operand, [rows, K] or [E, rows, K] of ``dtype`` (exact in bf16 and fp32; fp16 rounds, and
    overflows above 65504).  With offsets, rows behind the last expert's are zeros."""
    who = "mx.dequantize"
    _require(dtype in _DTYPES, f"{who}: dtype must be fp16, bf16 or fp32, got {dtype}")
    experts = None if offsets is None else _experts(who, offsets)
    matrices, rows, k = _check_operand(who, packed, scales, 2 if offsets is not None or packed.dim() != 3 else 3,
                                       experts)
    dev = _device(who, packed, scales, offsets)
    out = torch.empty((*packed.shape[:-1], k), dtype=dtype, device=packed.device)
    if out.numel():
        args = _lib.MxQuantArgs(out.data_ptr(), packed.data_ptr(), scales.data_ptr(),
                                None if offsets is None else offsets.data_ptr(), None, _DTYPES[dtype], rows, k,
                                matrices if experts is None else experts, 0, 0, k, rows * k, _raw_stream(dev))
        _lib.check(_lib.load().nvfp4_mx_dequantize(_byref(args)))
    return out


def _product(who, a, sa, b1, s1, b2, s2, offsets, out_dtype):
    _require(out_dtype in _DTYPES, f"{who}: out_dtype must be fp16, bf16 or fp32, got {out_dtype}")
    experts = None
    if offsets is not None:
        experts = _experts(who, offsets)
        _require(b1.dim() == 3 and b1.shape[0] == experts,
                 f"{who}: offsets of {experts} experts need weights [{experts}, N, K/2], got {tuple(b1.shape)}")
    _, rows, k = _check_operand(who, a, sa, 2, experts)
    for b, s in ((b1, s1), (b2, s2)):
        if b is not None:
            _, n, kb = _check_operand(who, b, s, 2 if experts is None else 3)
            _require(kb == k and b.shape == b1.shape, f"{who}: weights {tuple(b.shape)} do not fit tokens with K={k}"
                     + ("" if b is b1 else f" and weights {tuple(b1.shape)}"))
    dev = _device(who, a, sa, b1, s1, b2, s2, offsets)
    c = torch.empty((rows, n), dtype=out_dtype, device=a.device)
    if c.numel():
        args = _lib.MxGemmArgs(a.data_ptr(), b1.data_ptr(), None if b2 is None else b2.data_ptr(), sa.data_ptr(),
                               s1.data_ptr(), None if b2 is None else s2.data_ptr(), c.data_ptr(),
                               None if offsets is None else offsets.data_ptr(), rows, n, k, experts or 1,
                               _DTYPES[out_dtype], 0, n, _raw_stream(dev))
        _lib.check(_lib.load().nvfp4_mx_gemm(_byref(args)))
        _post()
    return c


def gemm(a, sa, b, sb, offsets: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [rows, K] times the transpose of b [N, K] -> [rows, N], for any number of rows.

    With offsets, the rows are sorted by expert, b is [experts, N, K] and each row meets its expert's matrix; rows
    behind the last expert's come out as zeros."""
    return _product("mx.gemm", a, sa, b, sb, None, None, offsets, out_dtype)


def dual_gemm(a, sa, b1, sb1, b2, sb2, offsets: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """silu(a . b1^T) * (a . b2^T), otherwise as gemm; both products stay in fp32."""
    return _product("mx.dual_gemm", a, sa, b1, sb1, b2, sb2, offsets, out_dtype)
