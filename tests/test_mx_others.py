"""Rows that no expert has, in front of the first offset and from the last on: zeros in values, untouched in codes,
whatever the result's memory held.  Through the C interface, into memory of the test's own."""
import ctypes

import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib, mx
from nvfp4_b200.mx import _DTYPES
from tests import mxref
from tests.test_mx_gemm import DTYPES, f64, gate_close, on_gpu, operand, same, weights_on_gpu

pytestmark = pytest.mark.gpu

# rows, offsets, N, K: tiles of one CTA and of pairs, K split in a cluster, rows of C of any width
CASES = [(300, [130, 165, 200], 72, 96), (300, [200, 200, 200], 72, 96), (300, [1, 4, 7], 65, 96),
         (300, [0, 0, 300], 33, 64), (40, [39, 39, 40], 64, 8192), (90, [5, 60, 66], 128, 16384),
         (1300, [100, 690, 1290], 4096, 96), (900, [64, 64, 700], 4093, 160), (3000, [1, 1500, 2999], 640, 64)]


def stream():
    return torch.cuda.current_stream().cuda_stream


def tokens(rows, offsets, k, g, low=126):
    """An operand of rows sorted by expert, and its values."""
    a = operand(rows, k, g, low, low + 3)
    at, _ = mxref.scale_rows(offsets)
    ops = on_gpu(a[0], a[1][offsets[0]:offsets[-1]], at, mx.scale_blocks(rows, len(offsets) - 1))
    return ops, mxref.decode(*a)


def products(x, offsets, bs, n):
    want = np.zeros((len(x), n))
    for lo, hi, b in zip(offsets[:-1], offsets[1:], bs):
        want[lo:hi] = x[lo:hi] @ mxref.decode(*b).T
    return want


def call(a, ws, out, code, off, rows, n, k, scales=None):
    b, b2 = ws[0], ws[1] if len(ws) > 1 else (None, None)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    args = _lib.MxGemmArgs(ptr(a[0]), ptr(b[0]), ptr(b2[0]), ptr(a[1]), ptr(b[1]), ptr(b2[1]), ptr(out), ptr(scales),
                           ptr(off), rows, n, k, off.numel() - 1, code, 0, n, stream())
    _lib.check(_lib.load().nvfp4_mx_gemm(ctypes.byref(args)))
    assert _lib.device_status(True) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,offsets,n,k", CASES)
def test_products(rows, offsets, n, k, dtype):
    g = np.random.RandomState(rows + n)
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    experts = len(offsets) - 1
    bs = [[operand(n, k, g) for _ in range(experts)] for _ in range(2)]
    ws = [weights_on_gpu(b) for b in bs]
    a, x = tokens(rows, offsets, k, g)
    c = torch.full((rows + 1, n), float("nan"), dtype=dtype, device="cuda")
    call(a, ws[:1], c, _DTYPES[dtype], off, rows, n, k)
    same(c[:rows], products(x, offsets, bs[0], n))
    assert c[rows].isnan().all()
    a, x = tokens(rows, offsets, k, g, 127 - int(np.log2(k) / 2) - 4)
    c.fill_(float("nan"))
    call(a, ws, c, _DTYPES[dtype], off, rows, n, k)
    lo, hi = offsets[0], offsets[-1]
    gate_close(c[lo:hi], *(products(x, offsets, b, n)[lo:hi] for b in bs))
    assert not c[:lo].any() and not c[hi:rows].any() and c[rows].isnan().all()


@pytest.mark.parametrize("rows,offsets,n,k", [c for c in CASES if c[2] % 32 == 0])
def test_codes(rows, offsets, n, k):
    g = np.random.RandomState(rows + n)
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    ws = [weights_on_gpu([operand(n, k, g) for _ in offsets[1:]]) for _ in range(2)]
    a, _ = tokens(rows, offsets, k, g, 127 - int(np.log2(k) / 2) - 4)
    codes = torch.full((rows + 1, n // 2), 0xa5, dtype=torch.uint8, device="cuda")
    scales = torch.empty((mx.scale_blocks(rows, 2), -(-n // 128), 32, 4, 4), dtype=torch.uint8, device="cuda")
    call(a, ws, codes, 3, off, rows, n, k, scales)
    lo, hi = offsets[0], offsets[-1]
    assert (codes[:lo] == 0xa5).all() and (codes[hi:] == 0xa5).all()
    values = mx.dual_gemm(*a, *ws[0], *ws[1], offsets=off, out_dtype=torch.float32)
    want = mx.dequantize(*mx.quantize(values, offsets=off), offsets=off, dtype=torch.float32)
    assert torch.equal(mx.dequantize(codes[:rows], scales, offsets=off, dtype=torch.float32), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,offsets,n,k", CASES)
def test_quantize_and_dequantize(rows, offsets, n, k, dtype):
    g = np.random.RandomState(rows)
    x = torch.from_numpy(g.randn(rows, k)).to(dtype)
    lo, hi = offsets[0], offsets[-1]
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    codes = torch.full((rows + 1, k // 2), 0xa5, dtype=torch.uint8, device="cuda")
    scales = torch.full((mx.scale_blocks(rows, 2), -(-k // 128), 32, 4, 4), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((rows + 1, k), float("nan"), dtype=dtype, device="cuda")
    xs = x.cuda()
    for name, t in (("nvfp4_mx_quantize", xs), ("nvfp4_mx_dequantize", out)):
        _lib.check(getattr(_lib.load(), name)(_lib.pack_mx_quant(
            t.data_ptr(), codes.data_ptr(), scales.data_ptr(), off.data_ptr(), 0, _DTYPES[dtype], rows, k, 2, 0, 0, k,
            0, stream())))
    assert (codes[:lo] == 0xa5).all() and (codes[hi:] == 0xa5).all()
    want = np.zeros((rows, k))
    want[lo:hi] = mxref.decode(*mxref.encode(f64(x)))[lo:hi]
    np.testing.assert_array_equal(f64(out[:rows]), want)
    assert out[rows].isnan().all()
