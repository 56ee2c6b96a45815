"""Rows between tokens and a part of the experts: offsets of some of them beside the slots of all.  Rows of other
experts are not read, come out as zeros wherever they lie, and are written by nobody else."""
import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib, moe
from nvfp4_b200.mx import _DTYPES
from tests.test_moe import DTYPES, f64, per_token, rows_case, within

pytestmark = pytest.mark.gpu

# tokens, top, experts, hidden, kind, first and last + 1 of the experts; each on the pack width that hidden allows, few
# slots (a CTA for each) and many (a warp)
PARTS = [(5, 8, 16, 64, "mixed", 3, 9), (33, 2, 4, 1023, "mixed", 2, 4), (7, 3, 5, 96, "mixed", 0, 2),
         (700, 2, 8, 512, "mixed", 2, 6), (900, 4, 9, 70, "mixed", 1, 9), (64, 6, 300, 38, "one", 0, 299),
         (64, 6, 300, 38, "one", 299, 300), (40, 3, 6, 32, "mixed", 3, 4)]


def part_of(case, dtype):
    """Lists, routing and their part; values with NaN where the part's rows are not."""
    tokens, top, experts, hidden, kind, first, last = case
    (order, slots, offsets), routing, x, ys, w = rows_case(tokens, top, experts, hidden, kind, dtype)
    lo, hi = int(offsets[first]), int(offsets[last])
    part = moe.Routing(routing.order, routing.slots, routing.offsets[first:last + 1])
    slots = np.where((slots >= lo) & (slots < hi), slots, -1)
    ys[:lo], ys[hi:] = float("nan"), float("nan")
    w[torch.from_numpy(slots < 0)] = float("nan")
    return order, slots, lo, hi, part, x.cuda(), ys.cuda(), w.cuda()


def call(name, routing, x, out, weights=None, grad=None, dweights=None):
    """A C entry point, into `out` and `dweights`, which hold NaN before."""
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    out.fill_(float("nan"))
    if dweights is not None:
        dweights.fill_(float("nan"))
    _lib.check(getattr(_lib.load(), name)(_lib.pack_moe(
        x.data_ptr(), ptr(grad), ptr(weights), out.data_ptr(), ptr(dweights), routing.slots.data_ptr(),
        routing.offsets.data_ptr(), _DTYPES[x.dtype], routing.tokens, routing.top, x.shape[1], routing.experts, 0,
        x.stride(0), 0 if grad is None else grad.stride(0), torch.cuda.current_stream().cuda_stream)))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", PARTS)
def test_rows_of_other_experts(dtype, case):
    order, slots, lo, hi, part, x, ys, w = part_of(case, dtype)
    tokens, top, _, hidden = case[:4]
    rows, own = tokens * top, order[lo:hi]
    clean = np.nan_to_num(f64(ys))
    weights = np.nan_to_num(f64(w))

    want = np.zeros((rows, hidden))
    want[lo:hi] = f64(x)[own // top]
    for _ in range(3):
        np.testing.assert_array_equal(f64(call("nvfp4_moe_gather", part, x, torch.empty_like(ys))), want)
    np.testing.assert_array_equal(f64(moe.gather(x, part)), want)

    # as for whole routings: `top` additions, or fused multiply-adds
    for got in (moe.gather_backward(ys, part), call("nvfp4_moe_gather_backward", part, ys, torch.empty_like(x))):
        within(got, per_token(slots, clean), dtype, top)
    for got in (moe.combine(ys, w, part), call("nvfp4_moe_combine", part, ys, torch.empty_like(x), w)):
        within(got, per_token(slots, clean, weights), dtype, top)

    want = np.zeros((rows, hidden))
    want[lo:hi] = weights.reshape(-1)[own, None] * f64(x)[own // top]
    taken = np.where((slots >= 0)[..., None], clean[np.maximum(slots, 0)], 0.0)
    products = f64(x)[:, None] * taken
    dweights = torch.empty_like(w)
    dys = call("nvfp4_moe_combine_backward", part, ys, torch.empty_like(ys), w, x, dweights)
    for dys, dw in ((dys, dweights), moe.combine_backward(x, ys, w, part)):
        within(dys, (want, np.abs(want)), dtype, 1)
        assert not f64(dys)[:lo].any() and not f64(dys)[hi:].any()
        within(dw, (products.sum(-1), np.abs(products).sum(-1)), torch.float32, hidden + 1)
        assert not f64(dw)[slots < 0].any()


def test_parts_add_up():
    """The experts in two halves, as two ranks that share the slots would have them: every row is in one of them."""
    (_, _, offsets), routing, x, ys, w = rows_case(60, 4, 8, 128, "mixed", torch.float32)
    x, ys, w = x.cuda(), ys.cuda(), w.cuda()
    halves = [routing._replace(offsets=routing.offsets[a:b]) for a, b in ((0, 5), (4, 9))]
    assert [h.experts for h in halves] == [4, 4]
    assert torch.equal(sum(moe.gather(x, h) for h in halves), moe.gather(x, routing))
    got = [moe.combine_backward(x, ys, w, h) for h in halves]
    for a, b, want in zip(*got, moe.combine_backward(x, ys, w, routing)):
        assert torch.equal(a + b, want)


@pytest.mark.parametrize("offsets", [[-7, 20, 1 << 30], [90, 90, 20], [30, 60, 40], [1 << 30, 5, -1]])
def test_offsets_that_fall_or_leave_the_rows_stay_in_bounds(offsets):
    _, routing, x, ys, w = rows_case(30, 3, 6, 64, "one", torch.bfloat16)  # every row has a slot
    x, ys, w = x.cuda(), ys.cuda(), w.cuda()
    lo = min(max(offsets[0], 0), 90)
    hi = min(max(offsets[-1], lo), 90)
    part = routing._replace(offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
    whole = moe.gather(x, routing)
    whole[:lo], whole[hi:] = 0, 0
    assert torch.equal(call("nvfp4_moe_gather", part, x, torch.empty_like(ys)), whole)
    dw = torch.empty_like(w)
    dys = call("nvfp4_moe_combine_backward", part, ys, torch.empty_like(ys), w, x, dw)
    want, _ = moe.combine_backward(x, ys, w, routing)
    want[:lo], want[hi:] = 0, 0
    assert torch.equal(dys, want) and torch.isfinite(dw).all()
