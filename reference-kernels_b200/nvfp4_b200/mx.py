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
``moe.sort`` returns, or a part of them for some of the experts): ``packed``
holds all rows without gaps, ``scales`` has ``min(rows, experts) + rows//128``
row blocks, and each expert's rows begin a new one, the first expert's the
first.  Nothing here reads the offsets on the host.

Launches go to the current CUDA stream; nothing is synchronised, and everything
can be captured into a CUDA graph.

Codes carry no gradient, like the integers that torch converts to: quantize of a
tensor that requires grad is a constant to autograd, and so is what is computed
from it.  A gradient is a product of its own (quantize, axis=0).
"""
from __future__ import annotations

import torch

from . import _lib
from .inputs import FP4X2
from .ops import _CHECK_STATUS, _post

E8M0 = torch.float8_e8m0fnu
_CODES = (FP4X2, torch.uint8)
_SCALES = (E8M0, torch.uint8)
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _fail(msg: str):
    """Calls of a few microseconds of GPU time are paced by the host: checks here test first and format their
    message (which takes longer than the test) only when they fail."""
    raise _lib.Nvfp4Error(msg)


def _device(who: str, t: torch.Tensor, *others) -> int:
    """The device of every tensor (None: not given), which has to be the current one."""
    dev = t.get_device()
    if dev < 0:
        _fail(f"{who}: expected a CUDA tensor (no CPU fallback)")
    for o in others:
        if o is not None and o.get_device() != dev:
            _fail(f"{who}: tensors on different devices (cuda:{dev} and {o.device})")
    if dev != _current_device():
        _fail(f"{who}: the tensors are on cuda:{dev} but cuda:{_current_device()} is current; "
              f"call inside torch.cuda.device({dev})")
    return dev


def _experts(who: str, offsets: torch.Tensor) -> int:
    if not (offsets.dtype is torch.int32 and offsets.dim() == 1 and 2 <= offsets.shape[0] <= 1025
            and offsets.is_contiguous()):
        _fail(f"{who}: offsets must be a contiguous int32 [experts + 1], at most 1024 experts")
    return offsets.shape[0] - 1


def scale_blocks(rows: int, experts: int | None = None) -> int:
    """Row blocks of the scales of ``rows`` rows (sorted by expert: for any offsets)."""
    return -(-rows // 128) if experts is None else min(rows, experts) + rows // 128


def _check_operand(who: str, packed: torch.Tensor, scales: torch.Tensor, dim: int, experts: int | None = None):
    """The shape of an operand's packed tensor; ``dim``: its dimensions; ``experts``: rows are sorted by expert."""
    shape = packed.shape
    if len(shape) != dim or packed.dtype not in _CODES or not packed.is_contiguous():
        _fail(f"{who}: codes must be contiguous float4_e2m1fn_x2 or uint8 of {dim} dimensions, "
              f"got {packed.dtype} {tuple(shape)} (strides {packed.stride()})")
    k2 = shape[-1]
    if k2 == 0 or k2 % 16:
        _fail(f"{who}: K={2 * k2} must be a positive multiple of 32")
    want = (scale_blocks(shape[-2], experts), -(-k2 // 64), 32, 4, 4)
    if dim == 3:
        want = (shape[0], *want)
    if scales.shape != want or scales.dtype not in _SCALES or not scales.is_contiguous():
        _fail(f"{who}: scales must be contiguous float8_e8m0fnu or uint8 {want}, "
              f"got {scales.dtype} {tuple(scales.shape)} (strides {scales.stride()})")
    return shape


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

    offsets: the rows are sorted by expert.  Codes of rows that no expert has
    are not written."""
    who = "mx.quantize"
    code = _DTYPES.get(x.dtype)
    if code is None:
        _fail(f"{who}: x must be fp16, bf16 or fp32, got {x.dtype}")
    shape, strides = x.shape, x.stride()
    dim = len(shape)
    if dim != 2 and dim != 3:
        _fail(f"{who}: x must be [rows, K] or [experts, rows, K], got {tuple(shape)}")
    rows, k = shape[-2], shape[-1]
    columns = axis == 0 and dim == 2
    if not columns and axis != -1 and axis != dim - 1:
        _fail(f"{who}: axis={axis} must be the last, or 0 of a matrix")
    if k == 0 or (k % 32 and not columns):
        _fail(f"{who}: K={k} must be a positive multiple of 32")
    if strides[-1] != 1 and k != 1:
        _fail(f"{who}: x must have unit stride along K (strides {strides})")
    dev = _device(who, x, offsets)
    if columns:
        if offsets is not None:
            _fail(f"{who}: axis=0 takes no offsets")
        kt = -(-rows // 32) * 32
        packed = x.new_empty((k, kt // 2), dtype=FP4X2)
        scales = x.new_empty((-(-k // 128), -(-kt // 128), 32, 4, 4), dtype=E8M0)
        if rows:
            _launch("nvfp4_mx_quantize", x, packed, scales, None, None, code, rows, k, 1, 0, 1, strides[0], 0, dev)
        return packed, scales
    experts = None
    if offsets is not None:
        if dim != 2:
            _fail(f"{who}: offsets need x [rows, K]")
        experts = _experts(who, offsets)
    blocks = (scale_blocks(rows, experts), -(-k // 128), 32, 4, 4)
    if dim == 2:
        packed = x.new_empty((rows, k // 2), dtype=FP4X2)
        scales = x.new_empty(blocks, dtype=E8M0)
        if rows:
            _launch("nvfp4_mx_quantize", x, packed, scales, offsets, None, code, rows, k, experts or 1, 0, 0,
                    strides[0], 0, dev)
    else:
        packed = x.new_empty((shape[0], rows, k // 2), dtype=FP4X2)
        scales = x.new_empty((shape[0], *blocks), dtype=E8M0)
        if rows and shape[0]:
            _launch("nvfp4_mx_quantize", x, packed, scales, None, None, code, rows, k, shape[0], 0, 0, strides[1],
                    strides[0], dev)
    return packed, scales


def _launch(name, x, packed, scales, offsets, slots, dtype, rows, k, experts, top, columns, rstride, estride, dev):
    """nvfp4_mx_quantize or nvfp4_mx_dequantize."""
    rc = getattr(_lib.load(), name)(_lib.pack_mx_quant(
        x.data_ptr(), packed.data_ptr(), scales.data_ptr(), 0 if offsets is None else offsets.data_ptr(),
        0 if slots is None else slots.data_ptr(), dtype, rows, k, experts, top, columns, rstride, estride,
        _raw_stream(dev)))
    if rc:
        _lib.check(rc)


def dequantize(packed: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an operand, [rows, K] or [E, rows, K] of ``dtype`` (exact in bf16 and fp32; fp16 rounds, and
    overflows above 65504).  With offsets, rows that no expert has are zeros."""
    who = "mx.dequantize"
    code = _DTYPES.get(dtype)
    if code is None:
        _fail(f"{who}: dtype must be fp16, bf16 or fp32, got {dtype}")
    experts = None if offsets is None else _experts(who, offsets)
    shape = _check_operand(who, packed, scales, 3 if experts is None and packed.dim() == 3 else 2, experts)
    dev = _device(who, packed, scales, offsets)
    rows, k = shape[-2], 2 * shape[-1]
    out = packed.new_empty((*shape[:-1], k), dtype=dtype)
    if out.numel():
        if experts is None:
            experts = shape[0] if len(shape) == 3 else 1
        _launch("nvfp4_mx_dequantize", out, packed, scales, offsets, None, code, rows, k, experts, 0, 0, k, rows * k,
                dev)
    return out


def _product(who, a, sa, b1, s1, b2, s2, offsets, out_dtype, quantize=False):
    code = 3 if quantize else _DTYPES.get(out_dtype)
    if code is None:
        _fail(f"{who}: out_dtype must be fp16, bf16 or fp32, got {out_dtype}")
    experts, dim = None, 2
    if offsets is not None:
        experts, dim = _experts(who, offsets), 3
        if b1.dim() != 3 or b1.shape[0] != experts:
            _fail(f"{who}: offsets of {experts} experts need weights [{experts}, N, K/2], got {tuple(b1.shape)}")
    rows, k2 = _check_operand(who, a, sa, 2, experts)
    shape = _check_operand(who, b1, s1, dim)
    if shape[-1] != k2:
        _fail(f"{who}: weights {tuple(shape)} do not fit tokens with K={2 * k2}")
    if b2 is not None and _check_operand(who, b2, s2, dim) != shape:
        _fail(f"{who}: weights {tuple(b2.shape)} do not fit weights {tuple(shape)}")
    dev = _device(who, a, sa, b1, s1, b2, s2, offsets)
    n = shape[-2]
    if quantize:
        if n == 0 or n % 32:
            _fail(f"{who}: N={n} must be a positive multiple of 32 for a quantised result")
        c = a.new_empty((rows, n // 2), dtype=FP4X2)
        sc = a.new_empty((scale_blocks(rows, experts), -(-n // 128), 32, 4, 4), dtype=E8M0)
    else:
        c, sc = a.new_empty((rows, n), dtype=out_dtype), None
    if rows and n:
        gated = b2 is not None
        rc = _lib.load().nvfp4_mx_gemm(_lib.pack_mx_gemm(
            a.data_ptr(), b1.data_ptr(), b2.data_ptr() if gated else 0, sa.data_ptr(), s1.data_ptr(),
            s2.data_ptr() if gated else 0, c.data_ptr(), sc.data_ptr() if quantize else 0,
            0 if offsets is None else offsets.data_ptr(), rows, n, 2 * k2, experts or 1, code, 0, n, _raw_stream(dev)))
        if rc:
            _lib.check(rc)
        if _CHECK_STATUS:
            _post()
    return (c, sc) if quantize else c


def gemm(a, sa, b, sb, offsets: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [rows, K] times the transpose of b [N, K] -> [rows, N], for any number of rows.

    With offsets, the rows are sorted by expert, b is [experts, N, K] and each row meets its expert's matrix; rows
    that no expert has come out as zeros."""
    return _product("mx.gemm", a, sa, b, sb, None, None, offsets, out_dtype)


def dual_gemm(a, sa, b1, sb1, b2, sb2, offsets: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
              quantize: bool = False):
    """silu(a . b1^T) * (a . b2^T), otherwise as gemm; both products stay in fp32.

    quantize=True (N % 32 == 0): the result as an MXFP4 operand (packed, scales), quantised from fp32 in the product's
    epilogue: what mx.quantize of the fp32 result, with the same offsets, gives."""
    return _product("mx.dual_gemm", a, sa, b1, sb1, b2, sb2, offsets, out_dtype, quantize)
