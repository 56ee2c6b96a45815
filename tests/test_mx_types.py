"""Operands are codes and scales of their own types, or bytes; other types of one byte hold values of other formats."""
import pytest
import torch

from nvfp4_b200 import _lib, mx

CODES = [torch.float4_e2m1fn_x2, torch.uint8]
SCALES = [torch.float8_e8m0fnu, torch.uint8]
ONE_BYTE = [torch.float4_e2m1fn_x2, torch.float8_e8m0fnu, torch.uint8, torch.int8, torch.bool, torch.float8_e4m3fn,
            torch.float8_e5m2]


def calls(codes, scales):
    a, sa = torch.zeros((8, 32), dtype=torch.uint8), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8)
    p, s = a.view(codes), sa.view(scales)
    return [lambda: mx.dequantize(p, s), lambda: mx.gemm(p, s, a, sa), lambda: mx.gemm(a, sa, p, s),
            lambda: mx.dual_gemm(a, sa, a, sa, p, s)]


@pytest.mark.parametrize("dtype", ONE_BYTE)
def test_types(dtype):
    for call in calls(dtype, torch.uint8):
        with pytest.raises(_lib.Nvfp4Error, match="CUDA" if dtype in CODES else "codes must be"):
            call()
    for call in calls(torch.uint8, dtype):
        with pytest.raises(_lib.Nvfp4Error, match="CUDA" if dtype in SCALES else "scales must be"):
            call()
