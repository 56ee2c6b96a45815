"""Tokens sorted by expert and back: routing against a plain stable sort, rows,
sums and gradients against their formulas in 64 bits."""
import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib, moe, mx
from tests import mxref

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def f64(t):
    return t.double().cpu().numpy()


def make_ids(tokens, top, experts, seed, kind="mixed"):
    g = np.random.RandomState(seed)
    if kind == "one":
        ids = np.full((tokens, top), experts - 1)
    elif kind == "none":
        ids = np.where(g.rand(tokens, top) < 0.5, -1, experts)
    else:  # some slots dropped, some of another rank, some repeated within a token
        ids = g.randint(-1, experts + 2, (tokens, top))
    return ids


def within(got, want, dtype, sums):
    """|got - want| <= half a step of the result's type, and of fp32 for each of the `sums` roundings (relative to the
    sum of the magnitudes added, `want[1]`)."""
    value, magnitude = want
    bound = torch.finfo(dtype).eps / 2 * np.abs(value) + sums * 2.0 ** -24 * magnitude * (1 + torch.finfo(dtype).eps)
    bound = bound + float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps / 2  # subnormal results
    d = np.abs(f64(got) - value)
    assert (d <= bound).all(), (d - bound).max()


# ---------------------------------------------------------------- CPU
def test_refusals():
    ids = torch.zeros((4, 2), dtype=torch.int64)
    with pytest.raises(_lib.Nvfp4Error, match="CUDA"):
        moe.sort(ids, 4)
    for bad, what in [(ids.float(), "int32 or int64"), (ids[:, 0], "tokens, top"), (ids.t(), "contiguous")]:
        with pytest.raises(_lib.Nvfp4Error, match=what):
            moe.sort(bad, 4)
    order, slots, offsets = (torch.zeros(s, dtype=torch.int32) for s in ((8,), (4, 2), (5,)))
    r = moe.Routing(order, slots, offsets)
    x, xs, w = torch.zeros((4, 16)), torch.zeros((8, 16)), torch.zeros((4, 2))
    with pytest.raises(_lib.Nvfp4Error, match="CUDA"):
        moe.gather(x, r)
    for call, what in [
            (lambda: moe.gather(xs, r), "must be \\[4, hidden\\]"),
            (lambda: moe.gather(x.double(), r), "fp16, bf16 or fp32"),
            (lambda: moe.gather(torch.zeros((16, 4)).t(), r), "unit stride"),
            (lambda: moe.gather(x, moe.Routing(order, slots.long(), offsets)), "slots"),
            (lambda: moe.gather(x, moe.Routing(order, slots, offsets[:1])), "offsets"),
            (lambda: moe.gather(x, moe.Routing(order, slots, offsets.long())), "offsets"),
            (lambda: r._replace(slots=slots[:, 0]), "slots"),
            (lambda: moe.gather_backward(x, r), "must be \\[8, hidden\\]"),
            (lambda: moe.combine(xs, w.half(), r), "weights"),
            (lambda: moe.combine(xs, w[:, :1], r), "weights"),
            (lambda: moe.combine_backward(x.half(), xs, w, r), "type and hidden"),
            (lambda: moe.combine_backward(x[:, :8], xs, w, r), "type and hidden"),
            (lambda: moe.quantize_tokens(x, r), "multiple of 32")]:
        with pytest.raises(_lib.Nvfp4Error, match=what):
            call()


def test_c_refusals():
    import ctypes
    lib = _lib.load()
    fake = 1 << 20
    assert lib.nvfp4_moe_sort(fake, 2, 4, 4, fake, fake, fake, None, 0, None) == 1
    assert lib.nvfp4_moe_sort(fake, 4, -1, 4, fake, fake, fake, None, 0, None) == 1
    assert lib.nvfp4_moe_sort(fake, 4, 4, 0, fake, fake, fake, None, 0, None) == 1
    assert lib.nvfp4_moe_sort(fake, 4, 4, 1025, fake, fake, fake, None, 0, None) == 1
    assert lib.nvfp4_moe_sort(None, 4, 4, 4, fake, fake, fake, None, 0, None) == 3
    assert lib.nvfp4_moe_sort(fake, 4, 4, 4, fake, fake, None, None, 0, None) == 3
    assert lib.nvfp4_moe_sort(fake + 4, 8, 4, 4, fake, fake, fake, None, 0, None) == 2
    d = dict(out=fake, slots=fake, offsets=fake, weights=fake, dweights=fake, grad=fake, dtype=1, tokens=4, top=2,
             hidden=8, experts=4, in_stride=8, grad_stride=8)

    def rc(fn, **kw):
        a = _lib.MoeArgs(**{**d, "in_": fake, **kw})
        return getattr(lib, "nvfp4_moe_" + fn)(ctypes.byref(a))

    assert lib.nvfp4_moe_gather(None) == 3
    assert rc("gather", dtype=5) == 1 and rc("gather", tokens=-1) == 1 and rc("gather", experts=0) == 1
    assert rc("gather", tokens=1 << 30, top=4) == 1
    assert rc("gather", in_=None) == 3 and rc("gather", slots=None) == 3 and rc("gather", offsets=None) == 3
    assert rc("combine", weights=None) == 3 and rc("combine_backward", dweights=None) == 3
    assert rc("combine_backward", grad=None) == 3 and rc("combine", in_=fake + 1) == 2


# ---------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,top,experts,kind", [
    (1, 1, 1, "mixed"), (1, 8, 256, "mixed"), (7, 3, 5, "none"), (33, 2, 8, "one"), (201, 4, 1024, "mixed"),
    (1025, 4, 33, "mixed"), (3001, 2, 64, "mixed"), (8192, 4, 128, "mixed"), (5000, 3, 1000, "one"),
    (70001, 8, 7, "mixed")])
def test_sort(id_dtype, tokens, top, experts, kind):
    ids = make_ids(tokens, top, experts, tokens + top, kind)
    got = moe.sort(torch.from_numpy(ids).to(id_dtype).cuda(), experts)
    for g, w, name in zip(got, mxref.route(ids, experts), got._fields):
        assert g.dtype == torch.int32
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)


@pytest.mark.gpu
def test_sort_far_ids_and_empty():
    ids = torch.tensor([[2 ** 40, 1], [-2 ** 62, 0], [2 ** 32, 2 ** 32 + 1]], device="cuda")
    r = moe.sort(ids, 2)
    assert r.order.tolist() == [3, 1, -1, -1, -1, -1] and r.offsets.tolist() == [0, 1, 2]
    assert r.slots.tolist() == [[-1, 1], [-1, 0], [-1, -1]]
    for shape in ((0, 4), (4, 0)):
        r = moe.sort(torch.zeros(shape, dtype=torch.int64, device="cuda"), 3)
        assert r.offsets.tolist() == [0, 0, 0, 0] and r.order.numel() == 0
        x = torch.ones((shape[0], 64), device="cuda")
        assert moe.gather(x, r).shape == (0, 64)
        w = torch.zeros(shape, device="cuda")
        xs = torch.ones((0, 64), device="cuda")
        assert not moe.combine(xs, w, r).any() and not moe.gather_backward(xs, r).any()
        dys, dw = moe.combine_backward(x, xs, w, r)
        assert dys.shape == (0, 64) and dw.shape == shape
        assert moe.quantize_tokens(x, r)[0].shape == (0, 32)


ROWS = [(1, 1, 1, 8, "mixed"), (5, 8, 16, 64, "mixed"), (33, 2, 4, 1023, "mixed"), (7, 3, 5, 96, "none"),
        (130, 4, 9, 4100, "mixed"), (64, 6, 300, 38, "one"), (19, 40, 8, 2, "mixed"), (700, 2, 8, 4096, "mixed")]


def rows_case(tokens, top, experts, hidden, kind, dtype, seed=1):
    ids = make_ids(tokens, top, experts, seed, kind)
    g = torch.Generator().manual_seed(seed)
    routing = moe.sort(torch.from_numpy(ids).cuda(), experts)
    rand = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return (mxref.route(ids, experts), routing, rand(tokens, hidden).to(dtype), rand(tokens * top, hidden).to(dtype),
            rand(tokens, top))


def per_token(slots, rows, weights=None):
    """(sum, sum of magnitudes) of each token's rows."""
    here = (slots >= 0)[..., None]
    taken = np.where(here, rows[np.maximum(slots, 0)], 0.0)
    if weights is not None:
        taken = taken * weights[..., None]
    return taken.sum(1), np.abs(taken).sum(1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROWS)
def test_rows_and_gradients(dtype, case):
    (order, slots, offsets), routing, x, ys, w = rows_case(*case, dtype)
    tokens, top, experts, hidden, _ = case
    n = offsets[-1]
    xs = moe.gather(x.cuda(), routing)
    want = np.zeros((tokens * top, hidden))
    want[:n] = f64(x)[order[:n] // top]
    np.testing.assert_array_equal(f64(xs), want)
    # `top` fp32 additions
    within(moe.gather_backward(ys.cuda(), routing), per_token(slots, f64(ys)), dtype, top)
    # each fused multiply-add rounds once
    within(moe.combine(ys.cuda(), w.cuda(), routing), per_token(slots, f64(ys), f64(w)), dtype, top)
    dy = x
    dys, dw = moe.combine_backward(dy.cuda(), ys.cuda(), w.cuda(), routing)
    want = np.zeros((tokens * top, hidden))
    want[:n] = f64(w).reshape(-1)[order[:n], None] * f64(dy)[order[:n] // top]
    within(dys, (want, np.abs(want)), dtype, 1)
    taken = np.where((slots >= 0)[..., None], f64(ys)[np.maximum(slots, 0)], 0.0)
    products = f64(dy)[:, None] * taken
    # any order of adding `hidden` products
    within(dw, (products.sum(-1), np.abs(products).sum(-1)), torch.float32, hidden + 1)
    assert not f64(dw)[slots < 0].any()


@pytest.mark.gpu
def test_gradients_against_differences():
    """combine and gather are linear in each argument: a step of 1 along a direction gives the gradient's product with
    it, in fp32."""
    (order, slots, offsets), routing, x, ys, w = rows_case(23, 3, 6, 64, "mixed", torch.float32)
    x, ys, w = x.cuda(), ys.cuda(), w.cuda()
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda t: torch.randn(t.shape, generator=g, device="cuda")  # noqa: E731
    dy = rand(x)
    dys, dw = moe.combine_backward(dy, ys, w, routing)
    for name, grad, delta, call in [
            ("ys", dys, rand(ys), lambda d: moe.combine(d, w, routing)),
            ("weights", dw, rand(w), lambda d: moe.combine(ys, d, routing))]:
        moved = (call(delta).double() * dy.double()).sum().item()
        said = (grad.double() * delta.double()).sum().item()
        scale = (call(delta.abs()).abs().double() * dy.abs().double()).sum().item()
        assert abs(moved - said) <= 200 * 2.0 ** -24 * scale + 1e-12, name
    dxs, delta = rand(ys), rand(x)
    moved = (moe.gather(delta, routing).double() * dxs.double()).sum().item()
    said = (moe.gather_backward(dxs, routing).double() * delta.double()).sum().item()
    assert abs(moved - said) <= 4 * 2.0 ** -24 * (dxs.abs().double().sum().item() * 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_other_strides(dtype):
    (order, slots, offsets), routing, x, ys, w = rows_case(40, 3, 6, 70, "mixed", dtype)
    w = w.cuda()
    for a, b in ((1, 33), (2, 34), (8, 40)):
        xv, yv = x.cuda()[:, a:b], ys.cuda()[:, a:b]
        assert torch.equal(moe.gather(xv, routing), moe.gather(xv.contiguous(), routing))
        assert torch.equal(moe.gather_backward(yv, routing), moe.gather_backward(yv.contiguous(), routing))
        assert torch.equal(moe.combine(yv, w, routing), moe.combine(yv.contiguous(), w, routing))
        got, want = moe.combine_backward(xv, yv, w, routing), moe.combine_backward(xv.contiguous(), yv.contiguous(), w,
                                                                                  routing)
        assert torch.equal(got[0], want[0])
        within(got[1], (f64(want[1]), f64(want[1].abs()) + 64), torch.float32, 64)
    one = x.cuda()[:1].expand(40, 70)
    assert torch.equal(moe.gather(one, routing), moe.gather(one.contiguous(), routing))


@pytest.mark.gpu
def test_unrouted_rows_do_not_reach_results():
    """NaN in rows that no slot has, and NaN weights of unrouted slots, leave results as they are."""
    (order, slots, offsets), routing, x, ys, w = rows_case(50, 4, 5, 64, "mixed", torch.float32)
    n = int(offsets[-1])
    assert n < 200
    clean = moe.combine(ys.cuda(), w.cuda(), routing)
    ys[n:] = float("nan")
    w[torch.from_numpy(slots < 0)] = float("nan")
    assert torch.equal(moe.combine(ys.cuda(), w.cuda(), routing), clean)
    assert torch.isfinite(moe.gather_backward(ys.cuda(), routing)).all()
    dys, dw = moe.combine_backward(x.cuda(), ys.cuda(), w.cuda(), routing)
    assert torch.isfinite(dys).all() and torch.isfinite(dw).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,top,experts,hidden,kind", [
    (1, 1, 1, 32, "mixed"), (16, 8, 256, 7168, "mixed"), (9, 3, 4, 96, "none"), (300, 2, 3, 544, "one"),
    (77, 40, 1024, 160, "mixed")])
def test_quantize_tokens(dtype, tokens, top, experts, hidden, kind):
    """The same codes, scales and places as the quantised gathered rows."""
    (order, slots, offsets), routing, x, _, _ = rows_case(tokens, top, experts, hidden, kind, dtype)
    n = int(offsets[-1])
    packed, scales = moe.quantize_tokens(x.cuda(), routing)
    codes, sc = mxref.encode(f64(x))
    token = order[:n] // top
    np.testing.assert_array_equal(packed.view(torch.uint8).cpu().numpy()[:n], mxref.pack(codes)[token])
    at, _ = mxref.scale_rows(offsets)
    np.testing.assert_array_equal(mxref.plain_scales(scales.view(torch.uint8).cpu().numpy(), n, hidden, at), sc[token])
    values = mx.dequantize(packed, scales, offsets=routing.offsets, dtype=torch.float32)
    np.testing.assert_array_equal(f64(values)[:n], mxref.decode(codes, sc)[token])
    assert not f64(values)[n:].any()


@pytest.mark.gpu
def test_two_streams_and_graphs():
    """Long sorts (with a workspace) on two streams at once, and two captured ones replayed in turn."""
    all_ids = [make_ids(9000, 4, 64, s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in all_ids]
    dev = [torch.from_numpy(i).cuda() for i in all_ids]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, d in zip(streams, dev):
            with torch.cuda.stream(s):
                got.append(moe.sort(d, 64))
    torch.cuda.synchronize()
    want = [mxref.route(i, 64) for i in all_ids]
    for i, r in enumerate(got):
        for g, w in zip(r, want[i % 2]):
            np.testing.assert_array_equal(g.cpu().numpy(), w)
    graphs = []
    for d in dev:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = moe.sort(d, 64)
        graphs.append((g, out))
    for _ in range(2):
        for (g, out), w in zip(graphs, want):
            g.replay()
    torch.cuda.synchronize()
    for (g, out), w in zip(graphs, want):
        for a, b in zip(out, w):
            np.testing.assert_array_equal(a.cpu().numpy(), b)
