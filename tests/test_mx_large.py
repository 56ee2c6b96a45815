"""MXFP4 and expert operators on tensors of more than 2^32 elements, or 2^31 bytes per row: everything zero but the corners,
so that a wrapped address shows as a value that is missing or in the wrong place."""
import pytest
import torch

from nvfp4_b200 import _lib, moe, mx

pytestmark = pytest.mark.gpu


def corners(t):
    return t[[0, 0, -1, -1], [0, -1, 0, -1]].float().tolist()


def nonzero(t):
    """Elements of t that are not zero, a part at a time."""
    return sum(int(torch.count_nonzero(part)) for part in t.view(-1).split(1 << 29))


def operand(rows, k, codes=0x22):
    """`codes` (two e2m1 values, 1.0) in the first and the last row."""
    packed = torch.zeros((rows, k // 2), dtype=torch.uint8, device="cuda")
    packed[0] = packed[-1] = codes
    return packed, torch.full((mx.scale_blocks(rows), -(-k // 128), 32, 4, 4), 127, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("rows,n,dtype", [(1, 2 ** 29 + 40, torch.float32), (2, 2 ** 30 + 64, torch.bfloat16),
                                          (2 ** 17 + 5, 2 ** 15 + 24, torch.bfloat16),
                                          (2 ** 15 + 5, 2 ** 17 + 3, torch.float16)])
def test_gemm(rows, n, dtype):
    c = mx.gemm(*operand(rows, 32), *operand(n, 32), out_dtype=dtype)
    assert _lib.device_status(True) == 0
    assert corners(c) == [32.0] * 4 and nonzero(c) == (2 if rows == 1 else 4)


def test_quantized_result():
    rows, n = 2 ** 19 + 3, 2 ** 14 + 32
    b = operand(n, 32)
    packed, scales = mx.dual_gemm(*operand(rows, 32, 0x33), *b, *b, quantize=True)
    assert _lib.device_status(True) == 0
    packed = packed.view(torch.uint8)
    assert nonzero(packed) == 4
    # 48^2 (silu(48) is nearly 48) is 4.5 * 2^9: 4, code 6, in the first or the last nibble.
    assert [packed[i, j].item() for i in (0, -1) for j in (0, -1)] == [6, 6 << 4] * 2
    last = scales.view(torch.uint8)[(rows - 1) // 128, (n - 1) // 128, (rows - 1) % 32, (rows - 1) % 128 // 32,
                                    (n - 1) % 128 // 32].item()
    assert last == 127 + 9


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_and_back(dtype):
    rows, k = 2 ** 16 + 1, 2 ** 16 + 32
    x = torch.zeros((rows, k), dtype=dtype, device="cuda")
    x[0, 0] = x[0, -1] = x[-1, 0] = x[-1, -1] = 3
    packed, scales = mx.quantize(x)
    del x
    back = mx.dequantize(packed, scales, dtype=dtype)
    assert corners(back) == [3.0] * 4 and nonzero(back) == 4


def test_quantize_columns():
    rows, k = 2 ** 16 + 40, 2 ** 16 + 1
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    x[0, 0] = x[0, -1] = x[-1, 0] = x[-1, -1] = 3
    packed, scales = mx.quantize(x, axis=0)
    del x
    back = mx.dequantize(packed, scales)[:, :rows]
    assert corners(back) == [3.0] * 4 and int(torch.count_nonzero(back)) == 4


def test_rows():
    tokens, hidden = 2 ** 16 + 1, 2 ** 15 + 32
    ids = torch.zeros((tokens, 2), dtype=torch.int32, device="cuda")
    ids[:, 1] = 1
    routing = moe.sort(ids, 2)
    weights = torch.full((tokens, 2), 0.5, device="cuda")
    x = torch.zeros((tokens, hidden), dtype=torch.bfloat16, device="cuda")
    x[0, 0] = x[0, -1] = x[-1, 0] = x[-1, -1] = 3
    xs = moe.gather(x, routing)
    assert nonzero(xs) == 8 and corners(xs) == [3.0] * 4
    assert xs[tokens - 1:tokens + 1, 0].tolist() == [3.0, 3.0]
    y = moe.gather_backward(xs, routing)
    assert nonzero(y) == 4 and corners(y) == [6.0] * 4
    y = moe.combine(xs, weights, routing)
    assert nonzero(y) == 4 and corners(y) == [3.0] * 4
    del y
    dys, dweights = moe.combine_backward(x, xs, weights, routing)
    del xs
    assert nonzero(dys) == 8 and corners(dys) == [1.5] * 4
    assert dweights[[0, -1]].tolist() == [[18.0, 18.0]] * 2 and int(torch.count_nonzero(dweights)) == 4
    del dys
    packed, _ = moe.quantize_tokens(x, routing)
    assert nonzero(packed.view(torch.uint8)) == 8
