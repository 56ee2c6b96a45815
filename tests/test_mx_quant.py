"""MXFP4 quantiser and dequantiser: every result is exact, so codes, scales and
values equal the plain 64-bit form's bit for bit."""
import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib, mx
from tests import mxref

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def u8(t):
    return t.view(torch.uint8).cpu().numpy()


def f64(t):
    return t.double().cpu().numpy()


def sample(rows, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k), generator=g) * torch.exp2(torch.randint(-9, 9, (rows, 1), generator=g).float())
    return x.to(dtype)


# ---------------------------------------------------------------- CPU: the plain form and the refusals
def test_plain_form_known_block():
    x = np.zeros((1, 64))
    x[0, :8] = [6, 5, 2.5, -0.25, 0.26, -7.9, 3.5, 1.25]  # amax 7.9: scale 1
    x[0, 32] = 2.0 ** -140  # below the smallest scale's reach
    codes, scales = mxref.encode(x)
    assert scales.tolist() == [[127, 0]]
    assert codes[0, :8].tolist() == [7, 6, 4, 8, 1, 15, 6, 2]
    assert codes[0, 32] == 0
    np.testing.assert_array_equal(mxref.unpack(mxref.pack(codes)), codes)
    np.testing.assert_array_equal(mxref.plain_scales(mxref.blocked_scales(scales), 1, 64), scales)


def test_plain_form_bad_blocks():
    x = np.ones((1, 96))
    x[0, 3], x[0, 40] = np.nan, -np.inf
    codes, scales = mxref.encode(x)
    assert scales.tolist() == [[255, 255, 125]] and not codes[0, :64].any()
    assert np.isnan(mxref.decode(codes, scales)[0, :64]).all()


def test_refusals():
    x = torch.zeros((4, 64))
    with pytest.raises(_lib.Nvfp4Error, match="CUDA"):
        mx.quantize(x)
    for bad, what in [(x.double(), "fp16, bf16 or fp32"), (x[:, :48], "multiple of 32"), (x[0], "rows, K"),
                      (x.t(), "multiple of 32|stride"), (torch.zeros((64, 64)).t(), "stride"),
                      (torch.zeros((4, 0)), "multiple of 32")]:
        with pytest.raises(_lib.Nvfp4Error, match=what):
            mx.quantize(bad)
    with pytest.raises(_lib.Nvfp4Error, match="axis"):
        mx.quantize(x.view(1, 4, 64), axis=0)
    with pytest.raises(_lib.Nvfp4Error, match="int32"):
        mx.dequantize(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((2, 1, 32, 4, 4), dtype=torch.uint8),
                      offsets=torch.zeros(3))
    for packed, scales, what in [
            (torch.zeros((4, 24), dtype=torch.uint8), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8), "multiple"),
            (torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 2, 32, 4, 4), dtype=torch.uint8), "scales"),
            (torch.zeros((4, 32)), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8), "codes"),
            (torch.zeros((32, 4), dtype=torch.uint8).t(), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8), "codes")]:
        with pytest.raises(_lib.Nvfp4Error, match=what):
            mx.dequantize(packed, scales)


def test_c_refusals():
    lib = _lib.load()
    fake = 1 << 20  # never dereferenced

    def args(**kw):
        d = dict(x=fake, packed=fake, scales=fake, dtype=1, rows=4, K=64, experts=1, x_rstride=64)
        return _lib.MxQuantArgs(**{**d, **kw})

    def rc(fn="nvfp4_mx_quantize", **kw):
        import ctypes
        return getattr(lib, fn)(ctypes.byref(args(**kw)))

    assert lib.nvfp4_mx_quantize(None) == 3
    assert rc(dtype=3) == 1 and rc(rows=-1) == 1 and rc(K=48) == 1 and rc(K=0) == 1 and rc(experts=0) == 1
    assert rc(x=None) == 3 and rc(scales=None) == 3
    assert rc(x=fake + 1) == 2 and rc(packed=fake + 8) == 2
    assert rc(offsets=fake, experts=1025) == 1 and rc(slots=fake) == 1
    assert rc(columns=1, experts=2) == 1 and rc(columns=1, offsets=fake) == 1
    assert rc(rows=1 << 30, experts=4) == 1
    assert rc("nvfp4_mx_dequantize", x=fake + 8) == 2 and rc("nvfp4_mx_dequantize", slots=fake, offsets=fake) == 1
    assert rc("nvfp4_mx_dequantize", columns=1) == 1


# ---------------------------------------------------------------- GPU
def check(x, packed, scales):
    """packed, scales are mx.quantize of x [rows, K]."""
    rows, k = x.shape
    codes, sc = mxref.encode(f64(x))
    np.testing.assert_array_equal(mxref.plain_scales(u8(scales), rows, k), sc)
    np.testing.assert_array_equal(u8(packed), mxref.pack(codes))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (130, 160), (128, 128), (257, 1024), (5, 7168), (2000, 544)])
def test_quantize_rows(dtype, rows, k):
    x = sample(rows, k, dtype, rows + k)
    x[0, :32] = 0
    packed, scales = mx.quantize(x.cuda())
    assert packed.dtype == torch.float4_e2m1fn_x2 and scales.dtype == torch.float8_e8m0fnu
    check(x, packed, scales)
    pad = u8(scales)[:, :, :, :, :][-1, -1, (rows - 1) % 32, ((rows - 1) % 128) // 32]
    assert not pad[(k // 32 - 1) % 4 + 1:].any()  # columns past K / 32 of a row
    values = mxref.decode(*mxref.encode(f64(x)))
    for out in DTYPES:
        got = mx.dequantize(packed, scales, dtype=out)
        assert got.dtype == out
        np.testing.assert_array_equal(f64(got), f64(torch.from_numpy(values).to(out)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_special_values(dtype):
    top = torch.finfo(dtype)
    rows = [torch.full((32,), v) for v in (0.0, -0.0, top.max, -top.max, top.tiny, top.tiny / 4, float("nan"),
                                           float("inf"), -float("inf"))]
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] * 2 + [-0.25, -0.75, -1.25, -1.75, -2.5, -3.5,
                                                                            -5.0, -7.0] * 2)
    rows += [ties * 2.0 ** e for e in (-12, -3, 0, 5)]
    nan_payload = torch.ones(32)
    nan_payload[31] = float("nan")
    rows.append(nan_payload)
    x = torch.stack(rows).to(dtype)
    if dtype != torch.float16:
        x = torch.cat([x, (ties * 2.0 ** -130).to(dtype)[None], (ties * 2.0 ** -125).to(dtype)[None],
                       (ties * 2.0 ** 124).to(dtype)[None]])
    packed, scales = mx.quantize(x.cuda())
    check(x, packed, scales)
    got = f64(mx.dequantize(packed, scales, dtype=torch.float32))
    np.testing.assert_array_equal(got, mxref.decode(*mxref.encode(f64(x))))
    # and down the columns
    packed, scales = mx.quantize(x.t().contiguous().cuda(), axis=0)
    check(x, packed, scales)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strides_and_unaligned_bases(dtype):
    rows, k = 70, 160
    store = sample(rows, k + 37, dtype, 5).cuda()
    for view in (store[:, 1:1 + k], store[:, 16:16 + k], store[::2, 3:3 + k], store[:1, :k].expand(rows, k)):
        check(view.cpu(), *mx.quantize(view))
    stack = sample(3 * 40, k + 8, dtype, 6).cuda().view(3, 40, k + 8)[:, 4:, 8:]
    packed, scales = mx.quantize(stack)
    for e in range(3):
        check(stack[e].cpu(), packed[e], scales[e])
    assert torch.equal(mx.dequantize(packed, scales)[1], mx.dequantize(packed[1], scales[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (33, 5), (300, 130), (256, 64), (31, 67), (1000, 192), (129, 1)])
def test_quantize_columns(dtype, rows, cols):
    x = sample(rows, cols, dtype, rows * cols)
    want = torch.zeros((cols, -(-rows // 32) * 32), dtype=dtype)
    want[:, :rows] = x.t()
    check(want, *mx.quantize(x.cuda(), axis=0))
    store = sample(rows, cols + 3, dtype, 9)
    want[:, :rows] = store[:, 3:].t()
    check(want, *mx.quantize(store.cuda()[:, 3:], axis=0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,tail", [([5], 0), ([0, 130, 0, 1, 128, 0], 0), ([0, 0, 0], 7), ([3, 300, 129], 50),
                                         ([1] * 300, 11), ([2] * 1024, 0)])
def test_quantize_sorted_rows(dtype, counts, tail):
    offsets = np.concatenate([[0], np.cumsum(counts)])
    rows, n, k = sum(counts) + tail, sum(counts), 96
    x = sample(rows, k, dtype, rows)
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    packed, scales = mx.quantize(x.cuda(), offsets=off)
    assert scales.shape[0] == min(rows, len(counts)) + rows // 128
    codes, sc = mxref.encode(f64(x))
    at, _ = mxref.scale_rows(offsets)
    np.testing.assert_array_equal(u8(packed)[:n], mxref.pack(codes)[:n])
    np.testing.assert_array_equal(mxref.plain_scales(u8(scales), n, k, at), sc[:n])
    got = f64(mx.dequantize(packed, scales, offsets=off, dtype=torch.float32))
    np.testing.assert_array_equal(got[:n], mxref.decode(codes, sc)[:n])
    assert not got[n:].any()


@pytest.mark.gpu
def test_offsets_that_fall_or_leave_the_rows_stay_in_bounds():
    """Offsets are the caller's data: whatever they hold, rows and blocks stay inside the buffers."""
    rows, k = 200, 64
    x = sample(rows, k, torch.bfloat16, 3).cuda()
    for offsets in ([0, 500, 10, 200], [-7, 100, 50, 1 << 30], [150, 150, 20, 0]):
        off = torch.tensor(offsets, dtype=torch.int32).cuda()
        packed, scales = mx.quantize(x, offsets=off)
        values = mx.dequantize(packed, scales, offsets=off)
        torch.cuda.synchronize()
        clamped = np.maximum.accumulate(np.clip(offsets, 0, rows))
        codes, sc = mxref.encode(f64(x))
        want = mxref.decode(codes, sc)
        want[:clamped[0]] = 0
        want[clamped[-1]:] = 0
        np.testing.assert_array_equal(f64(values), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_every_code_and_scale(dtype):
    """All 256 scales times all 16 codes: exact in bf16 and fp32 (down to 2^-128), correctly rounded in fp16."""
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 1, axis=1)
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    packed = torch.from_numpy(mxref.pack(codes)).cuda()
    blocked = torch.from_numpy(mxref.blocked_scales(scales)).cuda()
    got = mx.dequantize(packed, blocked, dtype=dtype)
    want = torch.from_numpy(mxref.decode(codes, scales))
    if dtype == torch.float16:
        want = want.float()  # 6 * 2^127 and the like are infinite in both
    np.testing.assert_array_equal(f64(got), f64(want.to(dtype)))


@pytest.mark.gpu
def test_empty():
    packed, scales = mx.quantize(torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda"))
    assert packed.shape == (0, 32) and scales.shape == (0, 1, 32, 4, 4)
    assert mx.dequantize(packed, scales).shape == (0, 64)
    packed, scales = mx.quantize(torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda"), axis=0)
    assert packed.shape == (64, 0) and scales.shape == (1, 0, 32, 4, 4)


@pytest.mark.gpu
def test_other_stream_and_graph():
    x = sample(300, 256, torch.bfloat16, 8)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        xs = x.cuda()
        check(x, *mx.quantize(xs))
    torch.cuda.synchronize()
    static = torch.zeros_like(x).cuda()
    mx.quantize(static)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mx.quantize(static)
    for seed in (1, 2):
        y = sample(300, 256, torch.bfloat16, seed)
        static.copy_(y)
        g.replay()
        check(y, *out)
