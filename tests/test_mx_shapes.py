"""Every tile shape and K split that a product can take, plain, gated and quantised, for one matrix and for experts,
against 64-bit products; and that the cases here reach all of them, whatever the launcher's rule becomes.

Inputs are as in test_mx_gemm: scales of three binades, so that fp32 holds every partial sum.  (Terms are multiples of
2^-4 with a standard deviation below 16, 2^24 of them 65536: over 500 standard deviations of a sum of 16384.)"""
import ctypes
import math

import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib, mx
from tests import mxref
from tests.test_mx_gemm import DTYPES, f64, gate_close, same_operand

SMS = 148

# (tokens of a tile, CTAs that share it, CTAs that share its K): all that the launcher has.
SHAPES = [(32, 1, 1), (32, 1, 2), (32, 1, 4), (32, 1, 8), (64, 1, 1), (64, 1, 2), (64, 1, 4), (64, 1, 8), (128, 1, 1),
          (128, 1, 2), (128, 1, 4), (128, 1, 8), (128, 2, 1), (192, 2, 1), (256, 2, 1)]

# shape, rows, N, K, experts (None: one matrix); on 148 SMs
PLAIN = [
    ((32, 1, 1), 4, 32, 1824, None), ((32, 1, 2), 2, 3775, 14144, None), ((32, 1, 4), 1, 33, 7744, None),
    ((32, 1, 8), 1, 32, 15136, None), ((64, 1, 1), 39, 35, 160, None), ((64, 1, 2), 133, 1847, 14752, None),
    ((64, 1, 4), 40, 33, 6080, None), ((64, 1, 8), 41, 38, 12384, None), ((128, 1, 1), 133, 6475, 160, None),
    ((128, 1, 2), 389, 1427, 14528, None), ((128, 1, 4), 129, 1160, 5952, None), ((128, 1, 8), 78, 518, 12288, None),
    ((128, 2, 1), 390, 2795, 6624, None), ((192, 2, 1), 264, 6776, 160, None), ((256, 2, 1), 591, 4617, 160, None),
    # ordinary projections
    ((32, 1, 2), 1, 7168, 16384, None), ((128, 1, 2), 128, 7168, 16384, None), ((128, 2, 1), 300, 4096, 7168, None),
    ((32, 1, 1), 5, 33, 1856, 3), ((32, 1, 2), 34, 32, 15488, 40), ((32, 1, 4), 2, 32, 7456, 3),
    ((32, 1, 8), 1, 32, 15488, 3), ((64, 1, 1), 68, 32, 160, 3), ((64, 1, 2), 387, 524, 15456, 3),
    ((64, 1, 4), 64, 34, 6144, 3), ((64, 1, 8), 66, 38, 12224, 3), ((128, 1, 1), 332, 2562, 160, 3),
    ((128, 1, 2), 471, 933, 14688, 3), ((128, 1, 4), 176, 138, 6080, 13), ((128, 1, 8), 128, 34, 12736, 8),
    ((128, 2, 1), 550, 1846, 6752, 3), ((192, 2, 1), 436, 3092, 160, 5), ((256, 2, 1), 1675, 1129, 160, 13)]
GATED = [
    ((32, 1, 1), 4, 32, 1824, None), ((32, 1, 2), 1, 1920, 14368, None), ((32, 1, 4), 1, 32, 7456, None),
    ((32, 1, 8), 1, 32, 15168, None), ((64, 1, 1), 40, 32, 160, None), ((64, 1, 2), 143, 928, 14784, None),
    ((64, 1, 4), 41, 32, 5984, None), ((64, 1, 8), 39, 32, 12128, None), ((128, 1, 1), 265, 1888, 160, None),
    ((128, 1, 2), 279, 992, 14592, None), ((128, 1, 4), 132, 640, 5952, None), ((128, 1, 8), 79, 288, 12736, None),
    ((128, 2, 1), 586, 928, 6464, None), ((192, 2, 1), 136, 4864, 160, None), ((256, 2, 1), 207, 4896, 160, None),
    ((32, 1, 1), 4, 32, 1824, 3), ((32, 1, 2), 33, 32, 14176, 40), ((32, 1, 4), 1, 32, 7456, 3),
    ((32, 1, 8), 1, 32, 15136, 3), ((64, 1, 1), 64, 32, 160, 3), ((64, 1, 2), 389, 320, 14112, 3),
    ((64, 1, 4), 73, 32, 5984, 3), ((64, 1, 8), 66, 32, 12064, 3), ((128, 1, 1), 396, 1120, 160, 3),
    ((128, 1, 2), 454, 544, 14464, 3), ((128, 1, 4), 147, 96, 5920, 13), ((128, 1, 8), 134, 32, 12448, 8),
    ((128, 2, 1), 814, 608, 6848, 3), ((192, 2, 1), 808, 1120, 160, 3), ((256, 2, 1), 408, 2592, 160, 3)]


def shape_of(rows, n, k, experts=None, gated=False, sms=SMS, **over):
    """(tokens of a tile, CTAs that share it, CTAs that share its K), or the error code."""
    fake = 1 << 20
    args = dict(b2=fake if gated else None, offsets=fake if experts else None, rows=rows, N=n, K=k,
                experts=experts or 1, out_dtype=1, ldc=max(n, 1))
    out = [ctypes.c_int32() for _ in range(3)]
    rc = _lib.load().nvfp4_mx_gemm_shape(ctypes.byref(_lib.MxGemmArgs(**{**args, **over})), sms, *map(ctypes.byref, out))
    return rc if rc else tuple(v.value for v in out)


# ---------------------------------------------------------------- CPU
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sorted_rows", [False, True])
def test_cases_reach_every_shape(gated, sorted_rows):
    cases = [c for c in (GATED if gated else PLAIN) if (c[4] is not None) == sorted_rows]
    for case in cases:
        assert shape_of(*case[1:], gated=gated) == case[0], case
    assert {c[0] for c in cases} == set(SHAPES)


def test_there_are_no_other_shapes():
    """Sizes all over the range, in steps of a quarter of a binade."""
    step = [int(2 ** (i / 4)) for i in range(53)]
    found = {shape_of(rows, n, 32 * k, experts, gated) for rows in step[::2] for n in step[20::3] for k in step[:42:3]
             for experts in (None, 3, 16, 200) for gated in (False, True)}
    assert found <= set(SHAPES) and len(found) > 10


def test_shape_refusals():
    lib, fake = _lib.load(), 1 << 20
    out = ctypes.c_int32()
    assert lib.nvfp4_mx_gemm_shape(None, SMS, *[ctypes.byref(out)] * 3) == 3
    args = _lib.MxGemmArgs(rows=4, N=8, K=64, experts=1, out_dtype=1, ldc=8)
    assert lib.nvfp4_mx_gemm_shape(ctypes.byref(args), SMS, None, ctypes.byref(out), ctypes.byref(out)) == 3
    assert shape_of(0, 8, 64) == 1 and shape_of(4, 8, 48) == 1 and shape_of(4, 0, 64) == 1
    assert shape_of(4, 8, 64, sms=1) == 1 and shape_of(4, 8, 64, experts=1025) == 1
    assert shape_of(4, 8, 64, experts=2, offsets=None) == 3 and shape_of(4, 8, 64, gated=True, out_dtype=3) == 1
    assert shape_of(4, 32, 64, gated=True, out_dtype=3, c_scales=fake) == (64, 1, 1)


# ---------------------------------------------------------------- GPU
def operand(gen, rows, k, low=126):
    """Packed codes and scale bytes of three binades, on the GPU."""
    packed = torch.randint(0, 256, (rows, k // 2), generator=gen, dtype=torch.uint8, device="cuda")
    return packed, torch.randint(low, low + 3, (rows, k // 32), generator=gen, dtype=torch.uint8, device="cuda")


def stored(scales, at=None, blocks=None):
    """The stored order; padding is NaN."""
    return torch.from_numpy(mxref.blocked_scales(scales.cpu().numpy(), at, blocks, fill=255)).cuda()


def decode(packed, scales):
    """float64 values."""
    table = torch.tensor(np.concatenate([mxref.E2M1, -mxref.E2M1]), device="cuda")
    v = torch.stack([table[(packed & 15).long()], table[(packed >> 4).long()]], -1).view(packed.shape[0], -1)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)


def problem(case, matrices):
    """Operands of a case, the offsets or None, rows that an expert has, and the 64-bit product with each matrix."""
    shape, rows, n, k, experts = case
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert shape_of(*case[1:], gated=matrices == 2, sms=sms) == shape
    gen = torch.Generator(device="cuda").manual_seed(rows + n + k)
    low = 126 if matrices == 1 else 127 - int(math.log2(k) / 2) - 4  # the gate's argument spans its bend
    a = operand(gen, rows, k, low)
    if experts is None:
        bs = [operand(gen, n, k) for _ in range(matrices)]
        ops = [(a[0], stored(a[1]))] + [(p, stored(s)) for p, s in bs]
        return ops, None, rows, [(decode(*a) @ decode(*b).t()).cpu().numpy() for b in bs]
    g = np.random.RandomState(rows)
    used = rows - rows // 20
    cuts = np.sort(g.randint(0, used + 1, experts - 1))
    cuts[0] = 0  # an expert without rows
    offsets = np.concatenate([[0], cuts, [used]])
    at, _ = mxref.scale_rows(offsets)
    bs = [[operand(gen, n, k) for _ in range(experts)] for _ in range(matrices)]
    ops = [(a[0], stored(a[1][:used], at, mx.scale_blocks(rows, experts)))]
    ops += [(torch.stack([p for p, _ in ws]), torch.stack([stored(s) for _, s in ws])) for ws in bs]
    x, want = decode(*a), []
    for ws in bs:
        y = torch.zeros((rows, n), dtype=torch.float64, device="cuda")
        for lo, hi, w in zip(offsets[:-1], offsets[1:], ws):
            y[lo:hi] = x[lo:hi] @ decode(*w).t()
        want.append(y.cpu().numpy())
    return ops, torch.from_numpy(offsets.astype(np.int32)).cuda(), used, want


@pytest.mark.gpu
@pytest.mark.parametrize("case", PLAIN)
def test_plain(case):
    (a, b), offsets, _, (want,) = problem(case, 1)
    for dtype in DTYPES:
        got = mx.gemm(*a, *b, offsets=offsets, out_dtype=dtype)
        np.testing.assert_array_equal(f64(got), f64(torch.from_numpy(want).to(dtype)))
        assert torch.equal(got, mx.gemm(*a, *b, offsets=offsets, out_dtype=dtype))
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("case", GATED)
def test_gated_and_quantized(case):
    (a, b1, b2), offsets, used, (x1, x2) = problem(case, 2)
    for dtype in DTYPES:
        got = mx.dual_gemm(*a, *b1, *b2, offsets=offsets, out_dtype=dtype)
        gate_close(got[:used], x1[:used], x2[:used])
        assert not got[used:].any()
    codes = mx.dual_gemm(*a, *b1, *b2, offsets=offsets, quantize=True)
    at = np.arange(used) if offsets is None else mxref.scale_rows(offsets.tolist())[0]
    same_operand(codes, mx.quantize(got, offsets=offsets), case[1], at)  # (got: the fp32 result)
    assert _lib.device_status(True) == 0
