"""The MXFP4 operators together, as they are used: an expert MLP, and the three
products of a training step of one linear layer."""
import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib, moe, mx
from tests import mxref


def f64(t):
    return t.double().cpu().numpy()


def values(x):
    return mxref.decode(*mxref.encode(x))


def stacked(w):
    """mx.quantize of weights [E, N, K] and their values."""
    return mx.quantize(w.cuda()), np.stack([values(f64(one)) for one in w])


def test_refusals():
    x, w = torch.zeros((4, 32)), (torch.zeros((8, 16), dtype=torch.uint8),) * 2
    with pytest.raises(_lib.Nvfp4Error, match="gate"):
        moe.mlp(x, torch.zeros((4, 2), dtype=torch.int64), torch.zeros((4, 2)), w, w, w)


CASES = [(1, 2, 4, 64, 96), (40, 3, 5, 160, 128), (300, 2, 3, 256, 288), (17, 8, 64, 96, 64), (200, 4, 20, 512, 160)]


def layer(tokens, top, experts, hidden, inner, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, hidden), generator=g).to(dtype)
    ids = torch.randint(-1, experts + 1, (tokens, top), generator=g)  # some dropped, some of another rank
    weights = torch.rand((tokens, top), generator=g)
    gate, up = (stacked((torch.randn((experts, inner, hidden), generator=g) * hidden ** -0.5).to(dtype))
                for _ in range(2))
    down = stacked((torch.randn((experts, hidden, inner), generator=g) * inner ** -0.5).to(dtype))
    return x, ids, weights, gate, up, down


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES)
def test_mlp(dtype, case):
    """Against the 64-bit form of the same steps.  The gated values are rounded from fp32 to 4 bits, where a difference
    in their last places can move a value to the next magnitude of its block: at most a step of a third of the value,
    or of a twelfth of its block's largest, for a share of the values that their distance from the borders gives.  So the bound on a result is statistical: an error of that share of such steps, whose
    squares add up (here doubled), and never more than the sum of all of them."""
    tokens, top, experts, hidden, inner = case
    x, ids, weights, (gate, wg), (up, wu), (down, wd) = layer(*case, dtype, 7)
    y = moe.mlp(x.cuda(), ids.cuda(), weights.cuda(), gate, up, down)
    assert y.shape == x.shape and y.dtype == dtype
    xq = values(f64(x))
    want = np.zeros((tokens, hidden))
    for t in range(tokens):
        for j in range(top):
            e = int(ids[t, j])
            if 0 <= e < experts:
                a, b = wg[e] @ xq[t], wu[e] @ xq[t]
                h = values((a / (1 + np.exp(-a)) * b)[None])[0]
                want[t] += float(weights[t, j]) * f64((torch.from_numpy(wd[e] @ h)).to(dtype))
    eps = torch.finfo(dtype).eps
    # share of the values within 2^-18 of a border, which is more than the gate's fp32 error, against spacings of at
    # least 1/4 of the value; each moves by at most 1/3 of a value.  (One of the few hundred values of the smallest
    # case is a share of 1e-3.)
    share = max(8 * 2.0 ** -18, 1e-3)
    bound = 2 * np.sqrt(share) / 3 + 4 * eps
    error = np.linalg.norm(f64(y) - want) / max(np.linalg.norm(want), 1e-30)
    assert error <= bound, (error, bound)
    assert not f64(y)[~((ids >= 0) & (ids < experts)).any(1).numpy()].any()
    assert _lib.device_status(True) == 0


@pytest.mark.gpu
def test_mlp_steps_are_its_own_operators_and_it_can_be_captured():
    x, ids, weights, (gate, _), (up, _), (down, _) = layer(90, 3, 6, 128, 160, torch.bfloat16, 9)
    x, ids, weights = x.cuda(), ids.cuda(), weights.cuda()

    def steps(x, ids, weights):
        r = moe.sort(ids, 6)
        h = mx.dual_gemm(*mx.quantize(moe.gather(x, r), offsets=r.offsets), *gate, *up, offsets=r.offsets,
                         out_dtype=torch.float32)
        return moe.combine(mx.gemm(*mx.quantize(h, offsets=r.offsets), *down, offsets=r.offsets), weights, r)

    assert torch.equal(moe.mlp(x, ids, weights, gate, up, down), steps(x, ids, weights))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moe.mlp(x, ids, weights, gate, up, down)
    for seed in (3, 4):
        other = layer(90, 3, 6, 128, 160, torch.bfloat16, seed)
        x.copy_(other[0])
        ids.copy_(other[1])
        weights.copy_(other[2])
        graph.replay()
        assert torch.equal(y, steps(x, ids, weights))
    # an eager call on another stream while the graph lives
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = moe.mlp(x, ids, weights, gate, up, down)
    torch.cuda.synchronize()
    assert torch.equal(z, y)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,top", [(0, 2), (5, 0), (5, 2)])
def test_mlp_without_routed_tokens(tokens, top):
    _, _, _, (gate, _), (up, _), (down, _) = layer(1, 1, 3, 64, 96, torch.bfloat16, 2)
    x = torch.ones((tokens, 64), dtype=torch.bfloat16, device="cuda")
    ids = torch.full((tokens, top), -1, device="cuda")
    y = moe.mlp(x, ids, torch.ones((tokens, top), device="cuda"), gate, up, down)
    assert y.shape == (tokens, 64) and not y.any()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,n,k", [(70, 96, 64), (257, 130, 200), (512, 384, 256)])
def test_linear_layer_forward_and_gradients(tokens, n, k):
    """y = x w^T, dx = dy w, dw = dy^T x, each with both operands in MXFP4 along its own sum (axis=0 quantises along
    the rows): equal to the 64-bit products of the operands' values but for the fp32 sums and the final rounding."""
    g = torch.Generator().manual_seed(tokens)
    x, w, dy = (torch.randn(s, generator=g).to(torch.bfloat16) for s in ((tokens, k), (n, k), (tokens, n)))

    def along(t, axis):
        t = f64(t) if axis else f64(t).T
        return values(np.pad(t, ((0, 0), (0, -t.shape[1] % 32))))

    def operand(t, axis):
        t = t.cuda()
        if axis and t.shape[1] % 32:
            t = torch.nn.functional.pad(t, (0, -t.shape[1] % 32))
        return mx.quantize(t, axis=axis)

    for (a, axis_a), (b, axis_b) in [((x, 1), (w, 1)), ((dy, 1), (w, 0)), ((dy, 0), (x, 0))]:
        got = mx.gemm(*operand(a, axis_a), *operand(b, axis_b), out_dtype=torch.float32)
        p, q = along(a, axis_a), along(b, axis_b)
        want, magnitude = p @ q.T, np.abs(p) @ np.abs(q).T
        assert got.shape == want.shape
        # sums of at most 512 terms, each addition off by a unit of fp32
        assert (np.abs(f64(got) - want) <= p.shape[1] * 2.0 ** -23 * magnitude + 1e-30).all()
