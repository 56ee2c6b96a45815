"""Inputs that require grad: refused where a result without a graph would lose the gradient, and the row operators
as the two ends of a torch.autograd.Function."""
import pytest
import torch

from nvfp4_b200 import _lib, moe, mx


def lists(tokens=4, top=2, experts=4):
    return moe.Routing(*(torch.zeros(s, dtype=torch.int32) for s in ((tokens * top,), (tokens, top), (experts + 1,))))


@pytest.mark.parametrize("of", ["x", "ys", "weights", "mlp x", "mlp weights"])
def test_refused_while_grad_mode_is_on(of):
    r = lists()
    x, xs, w = torch.zeros((4, 32)), torch.zeros((8, 32)), torch.zeros((4, 2))
    operand = (torch.zeros((4, 32, 16), dtype=torch.uint8), torch.zeros((4, 1, 1, 32, 4, 4), dtype=torch.uint8))
    mlp = lambda: moe.mlp(x, r.slots, w, operand, operand, operand)  # noqa: E731
    needs, call = {"x": (x, lambda: moe.gather(x, r)), "ys": (xs, lambda: moe.combine(xs, w, r)),
                   "weights": (w, lambda: moe.combine(xs, w, r)), "mlp x": (x, mlp), "mlp weights": (w, mlp)}[of]
    with pytest.raises(_lib.Nvfp4Error, match="CUDA"):
        call()
    needs.requires_grad_()
    with pytest.raises(_lib.Nvfp4Error, match="requires grad"):
        call()
    with torch.no_grad(), pytest.raises(_lib.Nvfp4Error, match="CUDA"):
        call()
    with torch.inference_mode(), pytest.raises(_lib.Nvfp4Error, match="CUDA"):
        call()


class Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, routing):
        ctx.routing = routing
        return moe.gather(x, routing)

    @staticmethod
    def backward(ctx, dxs):
        return moe.gather_backward(dxs.contiguous(), ctx.routing), None


class Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weights, routing):
        ctx.routing = routing
        ctx.save_for_backward(ys, weights)
        return moe.combine(ys, weights, routing)

    @staticmethod
    def backward(ctx, dy):
        return *moe.combine_backward(dy.contiguous(), *ctx.saved_tensors, ctx.routing), None


@pytest.mark.gpu
def test_gradients_through_a_function():
    """Small whole numbers: every product and sum is exact, in any order."""
    g = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randint(-4, 5, s, generator=g).float().cuda()  # noqa: E731
    tokens, top, experts, hidden = 37, 3, 5, 64
    ids = torch.randint(-1, experts + 1, (tokens, top), generator=g).cuda()
    x, w, scale, dy = rand(tokens, hidden), rand(tokens, top), rand(experts, hidden), rand(tokens, hidden)
    for t in (x, w, scale):
        t.requires_grad_()
    routing = moe.sort(ids, experts)
    rows = torch.arange(tokens * top, device="cuda")
    expert = (rows[:, None] >= routing.offsets[1:]).sum(1).clamp(max=experts - 1)
    y = Combine.apply(Gather.apply(x, routing) * scale[expert], w, routing)
    got = torch.autograd.grad(y, (x, w, scale), dy)
    here = (ids >= 0) & (ids < experts)
    each = scale.double()[ids.clamp(0, experts - 1)] * x.double()[:, None] * here[..., None]
    plain = (w.double()[..., None] * each).sum(1)
    assert torch.equal(y.double(), plain)
    for a, b in zip(got, torch.autograd.grad(plain, (x, w, scale), dy.double())):
        assert torch.equal(a.double(), b.double())


@pytest.mark.gpu
def test_codes_are_constants():
    x = torch.ones((4, 64), device="cuda", requires_grad=True)
    packed, scales = mx.quantize(x)
    assert not packed.requires_grad and not mx.dequantize(packed, scales).requires_grad
    assert not mx.gemm(packed, scales, packed, scales).requires_grad
