"""Products of MXFP4 operands.  With scales of a few binades every partial sum
is a multiple of 2^-2 times a power of two and below 2^24 of them, so fp32 holds
it whatever the order of the additions: the products must then be the 64-bit
result rounded once, exactly."""
import ctypes

import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib, mx
from tests import mxref

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def f64(t):
    return t.double().cpu().numpy()


def operand(rows, k, g, low=126, high=129, fill=255):
    """codes, scale bytes; padding of the stored scales is 255 (NaN) to show that nobody reads it."""
    return g.randint(0, 16, (rows, k)).astype(np.uint8), g.randint(low, high, (rows, k // 32)).astype(np.uint8)


def on_gpu(codes, scales, at=None, blocks=None):
    return (torch.from_numpy(mxref.pack(codes)).cuda(),
            torch.from_numpy(mxref.blocked_scales(scales, at, blocks, fill=255)).cuda())


def weights_on_gpu(ops):
    parts = [on_gpu(*o) for o in ops]
    return torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])


def same(got, want):
    np.testing.assert_array_equal(f64(got), f64(torch.from_numpy(want).to(got.dtype)))


def gated(x1, x2):
    with np.errstate(over="ignore"):
        return x1 / (1 + np.exp(-x1)) * x2


def gate_close(got, x1, x2):
    """Half a step of the type, and of fp32: expf's 2 + 1.2 |x| units (its argument is scaled by log2 e in fp32), 2 of
    the quotient, 1 of the sum, half of the product, each of 2^-23."""
    want = gated(x1, x2)
    eps = torch.finfo(got.dtype).eps
    bound = np.abs(want) * (eps / 2 + (6 + 1.2 * np.abs(x1)) * 2.0 ** -23) + 1e-35 * np.abs(x2)
    bound = bound + float(torch.finfo(got.dtype).smallest_normal) * eps / 2
    d = np.abs(f64(got) - want)
    assert (d <= bound).all(), (d / np.maximum(bound, 1e-300)).max()


# ---------------------------------------------------------------- CPU
def test_refusals():
    a, sa = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8)
    b, sb = torch.zeros((8, 32), dtype=torch.uint8), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8)
    with pytest.raises(_lib.Nvfp4Error, match="CUDA"):
        mx.gemm(a, sa, b, sb)
    off = torch.zeros(3, dtype=torch.int32)
    for call, what in [
            (lambda: mx.gemm(a, sa, b, sb, out_dtype=torch.float64), "out_dtype"),
            (lambda: mx.gemm(a[:, :16].contiguous(), sa, torch.zeros((8, 48), dtype=torch.uint8), sb), "do not fit"),
            (lambda: mx.gemm(a, sa, b, sa[:0]), "scales"),
            (lambda: mx.gemm(a.float(), sa, b, sb), "codes"),
            (lambda: mx.gemm(a[:, ::2], sa, b, sb), "codes"),
            (lambda: mx.gemm(a, sa, b, sb, offsets=off), "2 experts"),
            (lambda: mx.gemm(a, sa, b.view(1, 8, 32), sb.view(1, 1, 1, 32, 4, 4)), "2 dimensions"),
            (lambda: mx.dual_gemm(a, sa, b, sb, b[:4], sb), "do not fit"),
            (lambda: mx.dual_gemm(*((torch.zeros((8, 32), dtype=torch.uint8), sb) * 3), quantize=True), "CUDA|N=8"),
            (lambda: mx.gemm(a, sa, b.view(2, 4, 32), sb.expand(2, 1, 1, 32, 4, 4).contiguous(), offsets=off),
             "scales")]:
        with pytest.raises(_lib.Nvfp4Error, match=what):
            call()


def test_c_refusals():
    lib, fake = _lib.load(), 1 << 20
    d = dict(a=fake, b=fake, sfa=fake, sfb=fake, c=fake, rows=4, N=8, K=64, experts=1, out_dtype=1, ldc=8)

    def rc(**kw):
        return lib.nvfp4_mx_gemm(ctypes.byref(_lib.MxGemmArgs(**{**d, **kw})))

    assert lib.nvfp4_mx_gemm(None) == 3
    assert rc(out_dtype=4) == 1 and rc(out_dtype=3) == 1 and rc(rows=-1) == 1
    codes = dict(out_dtype=3, b2=fake, sfb2=fake)
    assert rc(**codes) == 1 and rc(**codes, N=32) == 3 and rc(**codes, N=32, c_scales=fake + 8) == 2
    assert rc(**codes, N=32, c_scales=fake, c=fake + 8) == 2 and rc(N=0) == 1 and rc(K=48) == 1 and rc(K=0) == 1
    assert rc(experts=0) == 1 and rc(experts=1025, offsets=fake) == 1 and rc(ldc=7) == 1
    assert rc(rows=2 ** 31 - 1, N=2 ** 31 - 1, ldc=2 ** 31) == 1 and rc(K=1 << 25) == 1
    assert rc(experts=2) == 3 and rc(a=None) == 3 and rc(b2=fake) == 3 and rc(sfb2=fake) == 3
    assert rc(a=fake + 8) == 2 and rc(sfb=fake + 8) == 2 and rc(c=fake + 1) == 2 and rc(offsets=fake + 2) == 2


@pytest.mark.parametrize("over", [2 ** 31 - 1, 2 ** 31 - 2 ** 20])
def test_c_refuses_sizes_near_32_bits(over):
    """The kernels round sizes up and step past them in 32-bit integers."""
    lib, fake = _lib.load(), 1 << 20

    def rc(name, struct, **kw):
        return getattr(lib, name)(ctypes.byref(struct(**kw)))

    product = dict(a=fake, b=fake, sfa=fake, sfb=fake, c=fake, experts=1, out_dtype=1, K=32)
    assert rc("nvfp4_mx_gemm", _lib.MxGemmArgs, **product, rows=over, N=1, ldc=1) == 1
    assert rc("nvfp4_mx_gemm", _lib.MxGemmArgs, **product, rows=1, N=over, ldc=over) == 1
    x = dict(x=fake, packed=fake, scales=fake, dtype=1, x_rstride=64)
    up = -(-over // 32) * 32
    for name in ("nvfp4_mx_quantize", "nvfp4_mx_dequantize"):
        assert rc(name, _lib.MxQuantArgs, **x, rows=1, K=min(up, 2 ** 31 - 32), experts=1) == 1
    assert rc("nvfp4_mx_quantize", _lib.MxQuantArgs, **x, rows=1, K=over, experts=1, columns=1) == 1
    assert rc("nvfp4_mx_quantize", _lib.MxQuantArgs, **x, rows=1, K=32, top=over, slots=fake, offsets=fake,
              experts=4) == 1
    assert lib.nvfp4_moe_sort(fake, 4, over, 4, fake, fake, fake, fake, 1 << 30, None) == 1
    assert lib.nvfp4_moe_sort_workspace(over, 4) == -1
    row = dict(in_=fake, grad=fake, weights=fake, out=fake, dweights=fake, slots=fake, offsets=fake, dtype=1, experts=4)
    for name in ("gather", "gather_backward", "combine", "combine_backward"):
        for sizes in [(over, 1, 1), (1, over, 1), (1, 1, over), (over, 0, 1)]:
            tokens, top, hidden = sizes
            assert rc("nvfp4_moe_" + name, _lib.MoeArgs, **row, tokens=tokens, top=top, hidden=hidden) == 1, (name, sizes)


def test_struct_layout_matches_header(tmp_path):
    import os
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "nvfp4_b200.h")
    structs = {"nvfp4_mx_quant_args": _lib.MxQuantArgs, "nvfp4_mx_gemm_args": _lib.MxGemmArgs,
               "nvfp4_moe_args": _lib.MoeArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {f[0].rstrip("_")}));' for f in py._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True).stdout.split()]
    want = []
    for py in structs.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f[0]).offset for f in py._fields_]
    assert got == want


def test_packed_bytes_equal_the_structs():
    for py, pack, n in [(_lib.MxQuantArgs, _lib.pack_mx_quant, 14), (_lib.MxGemmArgs, _lib.pack_mx_gemm, 17),
                        (_lib.MoeArgs, _lib.pack_moe, 16)]:
        values = [3 * i + 1 for i in range(n)]
        assert bytes(py(*values)) == pack(*values)
        with pytest.raises(_lib.Nvfp4Error, match="32-bit"):
            pack(*[1 << 31] * n)


# ---------------------------------------------------------------- GPU: one matrix
SIZES = [(1, 1, 32), (1, 128, 256), (5, 7, 64), (31, 130, 96), (33, 64, 160), (64, 257, 1024), (100, 300, 544),
         (130, 128, 7168), (193, 200, 288), (256, 129, 512), (385, 640, 320), (1000, 384, 736), (2049, 72, 128),
         # few tiles and a long K: shared by the CTAs of a cluster
         (1, 128, 8192), (17, 300, 4096), (70, 130, 4096), (128, 128, 16384), (2, 4096, 1024 + 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gemm_is_exact(dtype, m, n, k):
    g = np.random.RandomState(m + n + k)
    a, b = operand(m, k, g), operand(n, k, g)
    want = mxref.decode(*a) @ mxref.decode(*b).T
    got = mx.gemm(*on_gpu(*a), *on_gpu(*b), out_dtype=dtype)
    assert got.shape == (m, n) and got.dtype == dtype
    same(got, want)
    assert torch.equal(got, mx.gemm(*on_gpu(*a), *on_gpu(*b), out_dtype=dtype))
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [s for s in SIZES if s[2] <= 8192])
def test_dual_gemm(dtype, m, n, k):
    g = np.random.RandomState(m + n + k)
    # a small enough that the gate's argument spans both sides of its bend
    low = 127 - int(np.log2(k) / 2) - 4
    a, b1, b2 = operand(m, k, g, low, low + 3), operand(n, k, g), operand(n, k, g)
    x = mxref.decode(*a)
    got = mx.dual_gemm(*on_gpu(*a), *on_gpu(*b1), *on_gpu(*b2), out_dtype=dtype)
    gate_close(got, x @ mxref.decode(*b1).T, x @ mxref.decode(*b2).T)
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(3, 4096), (40, 1024), (200, 512)])
def test_scales_over_their_range(m, k):
    """Scales of all binades: |error| <= the fp32 error of a sum of k terms in any order, each addition off by up to a
    whole step (the tensor core may cut instead of rounding)."""
    g = np.random.RandomState(k)
    a, b = operand(m, k, g, 60, 190), operand(96, k, g, 100, 150)
    x, w = mxref.decode(*a), mxref.decode(*b)
    want, magnitude = x @ w.T, np.abs(x) @ np.abs(w).T
    got = f64(mx.gemm(*on_gpu(*a), *on_gpu(*b), out_dtype=torch.float32))
    assert (np.abs(got - want) <= k * 2.0 ** -23 * magnitude).all()
    # and in practice far less: the largest terms decide
    assert np.median(np.abs(got - want) / magnitude) < 2.0 ** -22


@pytest.mark.gpu
def test_nan_blocks_reach_only_their_rows_and_columns():
    g = np.random.RandomState(4)
    m, n, k = 70, 150, 512
    a, b = operand(m, k, g), operand(n, k, g)
    a[1][13, 5] = 255
    b[1][77, 15] = 255
    got = f64(mx.gemm(*on_gpu(*a), *on_gpu(*b), out_dtype=torch.float32))
    bad = np.zeros((m, n), bool)
    bad[13], bad[:, 77] = True, True
    assert np.isnan(got[bad]).all()
    a[1][13, 5], b[1][77, 15] = 127, 127
    want = mxref.decode(*a) @ mxref.decode(*b).T
    np.testing.assert_array_equal(got[~bad], want[~bad])


# Every tile shape (the launcher takes the one with the shortest rounds): 64, 128, 128, 192 and 256 tokens, the last
# three on CTA pairs; whole tiles, ragged ends, and rows of C that are not 16-byte aligned.
TILES = [(250, 4096, 64), (600, 3712, 64), (400, 4096, 96), (600, 4090, 160), (590, 4096, 320), (1000, 4096, 64),
         (1013, 4093, 544)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", TILES)
def test_every_tile_shape(dtype, m, n, k):
    g = np.random.RandomState(m + n + k)
    a, b = operand(m, k, g), operand(n, k, g)
    x = mxref.decode(*a)
    x1 = x @ mxref.decode(*b).T
    ops = on_gpu(*a)
    same(mx.gemm(*ops, *on_gpu(*b), out_dtype=dtype), x1)
    # gated tiles have half as many features
    n //= 2
    low = 127 - int(np.log2(k) / 2) - 4
    a = (a[0], g.randint(low, low + 3, (m, k // 32)).astype(np.uint8))
    halves = [(t[:n], s[:n]) for t, s in (b, operand(n, k, g))]
    x = mxref.decode(*a)
    got = mx.dual_gemm(*on_gpu(*a), *on_gpu(*halves[0]), *on_gpu(*halves[1]), out_dtype=dtype)
    gate_close(got, x @ mxref.decode(*halves[0]).T, x @ mxref.decode(*halves[1]).T)
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("counts,tail", [([1000], 0), ([1000, 3, 250], 1), ([400], 7), ([130, 270, 0, 511], 0)])
def test_every_tile_shape_with_experts(counts, tail):
    n, k = 4096, 96
    a, (b,), offsets, (want,) = grouped(counts, tail, n, k, 3)
    same(mx.gemm(*a, *b, offsets=offsets), want)
    n = 2048
    a, (b1, b2), offsets, (x1, x2) = grouped(counts, tail, n, k, 4, both=True)
    got = mx.dual_gemm(*a, *b1, *b2, offsets=offsets)
    gate_close(got[:sum(counts)], x1[:sum(counts)], x2[:sum(counts)])
    assert not f64(got[sum(counts):]).any()
    assert _lib.device_status(True) == 0


# ---------------------------------------------------------------- GPU: experts
GROUPS = [([5], 0), ([0, 0, 0], 9), ([1, 0, 40, 0, 0, 3], 5), ([130, 1, 0, 127, 128, 129], 0), ([300, 0, 5], 20),
          ([2] * 64, 3), ([1000, 3, 250], 1), ([0] * 500 + [7] + [0] * 523, 2), ([33] * 12, 0), ([70, 65, 64, 100], 0)]


def grouped(counts, tail, n, k, seed, both=False):
    g = np.random.RandomState(seed)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    rows, used = sum(counts) + tail, sum(counts)
    low = 127 - int(np.log2(k) / 2) - 4 if both else 126
    a = operand(rows, k, g, low, low + 3)
    at, _ = mxref.scale_rows(offsets)
    ops = on_gpu(a[0], a[1][:used], at, min(rows, len(counts)) + rows // 128)
    bs = [[operand(n, k, g) for _ in counts] for _ in range(2 if both else 1)]
    x = mxref.decode(*a)
    want = [np.concatenate([x[lo:hi] @ mxref.decode(*w).T for lo, hi, w in zip(offsets[:-1], offsets[1:], ws)]
                           + [np.zeros((tail, n))]) for ws in bs]
    return ops, [weights_on_gpu(ws) for ws in bs], torch.tensor(offsets, dtype=torch.int32).cuda(), want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(136, 288), (65, 512), (128, 1024)])
@pytest.mark.parametrize("counts,tail", GROUPS)
def test_experts(dtype, counts, tail, n, k):
    if len(counts) > 100:
        n, k = 33, 64
    a, (b,), offsets, (want,) = grouped(counts, tail, n, k, 1)
    same(mx.gemm(*a, *b, offsets=offsets, out_dtype=dtype), want)
    a, (b1, b2), offsets, (x1, x2) = grouped(counts, tail, n, k, 2, both=True)
    got = mx.dual_gemm(*a, *b1, *b2, offsets=offsets, out_dtype=dtype)
    used = sum(counts)
    gate_close(got[:used], x1[:used], x2[:used])
    assert not f64(got[used:]).any()
    assert _lib.device_status(True) == 0


def same_operand(got, want, rows, at):
    """Two operands' codes and scales of the rows that an expert has."""
    used = len(at)
    assert got[0].dtype == torch.float4_e2m1fn_x2 and got[0].shape == want[0].shape and got[1].shape == want[1].shape
    assert torch.equal(got[0].view(torch.uint8)[:used], want[0].view(torch.uint8)[:used])
    n = 2 * got[0].shape[1]
    a, b = (mxref.plain_scales(o[1].view(torch.uint8).cpu().numpy(), used, n, at) for o in (got, want))
    np.testing.assert_array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 32, 64), (5, 96, 160), (33, 160, 96), (200, 96, 288), (17, 320, 4096),
                                   (1, 64, 16384), (70, 128, 8192), (128, 160, 16384), (250, 2048, 64), (600, 1856, 64),
                                   (400, 2048, 96), (600, 2048, 320), (1013, 2048, 544), (3000, 1056, 32)])
def test_quantized_result(m, n, k):
    """The codes and scales that mx.quantize gives for the fp32 result, on every tile shape and K split."""
    g = np.random.RandomState(m + n + k)
    low = 127 - int(np.log2(k) / 2) - 4
    a, b1, b2 = operand(m, k, g, low, low + 3), operand(n, k, g), operand(n, k, g)
    a[0][0] = 0  # a zero row: zero blocks
    if m > 4:
        a[1][3, 0] = 255  # a NaN row
        b1[1][40 % n, k // 32 - 1] = 255  # a NaN column: its block in every row
    ops = on_gpu(*a) + on_gpu(*b1) + on_gpu(*b2)
    same_operand(mx.dual_gemm(*ops, quantize=True), mx.quantize(mx.dual_gemm(*ops, out_dtype=torch.float32)), m,
                 np.arange(m))
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(96, 288), (128, 512), (2048, 96)])
@pytest.mark.parametrize("counts,tail", [c for c in GROUPS if len(c[0]) < 100])
def test_quantized_result_of_experts(counts, tail, n, k):
    if n == 2048 and len(counts) > 6:
        n = 320
    a, (b1, b2), offsets, _ = grouped(counts, tail, n, k, 5, both=True)
    at, _ = mxref.scale_rows(offsets.tolist())
    want = mx.quantize(mx.dual_gemm(*a, *b1, *b2, offsets=offsets, out_dtype=torch.float32), offsets=offsets)
    same_operand(mx.dual_gemm(*a, *b1, *b2, offsets=offsets, quantize=True), want, sum(counts) + tail, at)
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
def test_offsets_that_fall_or_leave_the_rows_stay_in_bounds():
    g = np.random.RandomState(8)
    rows, n, k, experts = 200, 72, 96, 3
    bs = [operand(n, k, g) for _ in range(experts)]
    weights = weights_on_gpu(bs)
    for offsets in ([0, 500, 10, 200], [150, 150, 20, 0], [0, 60, 40, 1 << 30]):
        clamped = np.maximum.accumulate(np.clip(offsets, 0, rows))
        a = operand(rows, k, g)
        at, _ = mxref.scale_rows(clamped)
        lo, hi = clamped[0], clamped[-1]
        ops = on_gpu(a[0], a[1][lo:hi], at, experts + rows // 128)
        got = mx.gemm(*ops, *weights, offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
        want = np.concatenate([mxref.decode(a[0][s:t], a[1][s:t]) @ mxref.decode(*w).T
                               for s, t, w in zip(clamped[:-1], clamped[1:], bs)])
        same(got[lo:hi], want)
        assert _lib.device_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lo,hi", [(130, 200), (200, 200), (1, 7)])
def test_rows_of_no_expert_are_zeros(lo, hi, dtype):
    """Offsets of some of the experts: rows of others lie in front and behind."""
    g = np.random.RandomState(9)
    rows, n, k, experts = 300, 72, 96, 2
    bs = [operand(n, k, g) for _ in range(experts)]
    a = operand(rows, k, g)
    offsets = [lo, (lo + hi) // 2, hi]
    at, _ = mxref.scale_rows(offsets)
    ops = on_gpu(a[0], a[1][lo:hi], at, mx.scale_blocks(rows, experts))
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    dirt = torch.full((rows, n), float("nan"), dtype=dtype, device="cuda")  # what the result's memory holds before
    del dirt
    got = mx.gemm(*ops, *weights_on_gpu(bs), offsets=off, out_dtype=dtype)
    want = np.zeros((rows, n))
    for s, t, w in zip(offsets[:-1], offsets[1:], bs):
        want[s:t] = mxref.decode(a[0][s:t], a[1][s:t]) @ mxref.decode(*w).T
    same(got, want)
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
def test_empty():
    b = torch.zeros((8, 32), dtype=torch.uint8, device="cuda")
    sb = torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8, device="cuda")
    assert mx.gemm(b[:0], sb[:0], b, sb).shape == (0, 8)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert mx.gemm(b[:0], sb[:0], b.view(2, 4, 32), torch.stack([sb, sb]), offsets=off).shape == (0, 4)


@pytest.mark.gpu
def test_two_streams_at_once_and_graphs():
    """Products need no workspace: two streams, and two graphs, run side by side."""
    g = np.random.RandomState(11)
    cases = []
    for m, n, k in ((3, 256, 4096), (500, 256, 512)):
        a, b = operand(m, k, g), operand(n, k, g)
        cases.append((on_gpu(*a) + on_gpu(*b), mxref.decode(*a) @ mxref.decode(*b).T))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = []
    for _ in range(4):
        for s, (ops, want) in zip(streams, cases):
            with torch.cuda.stream(s):
                outs.append((mx.gemm(*ops), want))
    torch.cuda.synchronize()
    for got, want in outs:
        same(got, want)
    graphs = []
    for ops, want in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mx.gemm(*ops)
        graphs.append((graph, out, want))
    for graph, out, _ in graphs:
        out.zero_()
    torch.cuda.synchronize()
    for s, (graph, out, want) in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for graph, out, want in graphs:
        same(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3000, 2100, 32), (3000, 2104, 288), (5000, 1000, 800), (700, 24, 64), (40, 8, 128),
                                   (9000, 130, 544)])
def test_more_tiles_than_sms_and_narrow_results(m, n, k):
    """Many tiles of one to four K tiles in turn on each SM, and results narrower than a store's box."""
    g = np.random.RandomState(m + n + k)
    a, b = operand(m, k, g), operand(n, k, g)
    same(mx.gemm(*on_gpu(*a), *on_gpu(*b)), mxref.decode(*a) @ mxref.decode(*b).T)
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,ldc,shift", [(70, 130, 256, 144, 0), (300, 64, 96, 72, 8), (33, 40, 64, 41, 1),
                                             (1000, 4096, 64, 4112, 8), (1, 128, 8192, 136, 0)])
def test_rows_of_c_apart(m, n, k, ldc, shift):
    """C as part of a wider matrix through the C ABI: what lies beside it stays as it was."""
    g = np.random.RandomState(m + n)
    a, b = operand(m, k, g), operand(n, k, g)
    (pa, sa), (pb, sb) = on_gpu(*a), on_gpu(*b)
    c = torch.full((m + 1, ldc), 7.0, dtype=torch.bfloat16, device="cuda")
    args = _lib.MxGemmArgs(pa.data_ptr(), pb.data_ptr(), None, sa.data_ptr(), sb.data_ptr(), None,
                           c.data_ptr() + 2 * shift, None, None, m, n, k, 1, 1, 0, ldc,
                           torch.cuda.current_stream().cuda_stream)
    _lib.check(_lib.load().nvfp4_mx_gemm(ctypes.byref(args)))
    flat = c.reshape(-1)[shift:shift + m * ldc].view(m, ldc)
    same(flat[:, :n], mxref.decode(*a) @ mxref.decode(*b).T)
    flat[:, :n] = 7.0
    assert (c == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 128, 8192), (300, 256, 512), (600, 4096, 96), (1000, 4096, 1024)])
def test_withheld_load_is_reported(monkeypatch, m, n, k):
    """A load that never comes ends in a status within the waits' limit, and the next call is right again."""
    g = np.random.RandomState(2)
    a, b = operand(m, k, g), operand(n, k, g)
    ops = on_gpu(*a) + on_gpu(*b)
    monkeypatch.setenv("NVFP4_FAULT_INJECT", "1")
    mx.gemm(*ops)
    torch.cuda.synchronize()
    monkeypatch.delenv("NVFP4_FAULT_INJECT")
    assert _lib.device_status(True) != 0
    same(mx.gemm(*ops), mxref.decode(*a) @ mxref.decode(*b).T)
    assert _lib.device_status(True) == 0
