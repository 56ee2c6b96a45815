"""Cases that time the MXFP4 operators (e2m1 values, one power-of-two scale per
32) and the mixture-of-experts operators around them, in plain torch and
through the framework's own entry points (``own``).

A case is a dict with ``op``:

  quantize  MXFP4 codes of a matrix and back to values (a 4-bit copy of an
            activation or a weight), blocks along the rows (axis 1) or down
            the columns (axis 0, the operand of a weight gradient)
  gemm      the product of two MXFP4 operands, any number of tokens
  experts   the product of tokens sorted by expert with each expert's weights,
            plain or gated (silu(x W1^T) * (x W2^T))
  dispatch  slots sorted by expert, and the tokens' codes laid out in that order
  combine   the experts' rows back to tokens, weighted
  train     dispatch and combine of a training step with their gradients, in
            the activations' own type
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the activations of four tokens, before a projection: latency
        {"name": "quantize_decode", "op": "quantize", "rows": 4, "cols": 7168, "dtype": "bf16", "axis": 1},
        # the activations of a long prompt or of a training batch
        {"name": "quantize_prefill", "op": "quantize", "rows": 8192, "cols": 7168, "dtype": "bf16", "axis": 1},
        # the transposed operand of a weight gradient, an odd number of tokens
        {"name": "quantize_columns", "op": "quantize", "rows": 4007, "cols": 7168, "dtype": "fp16", "axis": 0},
        # one token through the projection that the GEMV benchmark has
        {"name": "gemm_one_token", "op": "gemm", "m": 1, "n": 7168, "k": 16384, "dtype": "bf16"},
        # a ragged batch of tokens through the same projection
        {"name": "gemm_prefill", "op": "gemm", "m": 1000, "n": 7168, "k": 16384, "dtype": "bf16"},
        # decoding: few tokens for each of many experts, gate and up projections
        {"name": "experts_decode", "op": "experts", "tokens": 32, "top": 8, "experts": 64, "of": 64,
         "k": 4096, "n": 2048, "gated": True, "dtype": "bf16"},
        # a prompt: many tokens for each expert
        {"name": "experts_prefill", "op": "experts", "tokens": 4096, "top": 4, "experts": 16, "of": 16,
         "k": 4096, "n": 2048, "gated": True, "dtype": "bf16"},
        # decoding with many small experts
        {"name": "dispatch_decode", "op": "dispatch", "tokens": 16, "top": 8, "experts": 256, "of": 256,
         "hidden": 7168, "dtype": "bf16"},
        # a prompt on one of two ranks that share the experts: the other's slots are not routed here
        {"name": "dispatch_prefill", "op": "dispatch", "tokens": 8191, "top": 4, "experts": 64, "of": 128,
         "hidden": 4096, "dtype": "bf16"},
        {"name": "combine_decode", "op": "combine", "tokens": 16, "top": 8, "experts": 256, "of": 256,
         "hidden": 7168, "dtype": "bf16"},
        # a small training step in 32 bits, odd sizes
        {"name": "train_small", "op": "train", "tokens": 201, "top": 2, "experts": 8, "of": 8,
         "hidden": 1023, "dtype": "fp32"},
        # a training batch
        {"name": "train_batch", "op": "train", "tokens": 8192, "top": 4, "experts": 64, "of": 64,
         "hidden": 4096, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "gemm", "experts", "dispatch", "combine", "train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "quantize":
        axis = rng.choice([1, 0])
        return {"op": op, "rows": _spread(rng, 1, 8192), "cols": 32 * _spread(rng, 4, 224), "dtype": dtype,
                "axis": axis}
    if op == "gemm":
        return {"op": op, "m": _spread(rng, 1, 2048), "n": _spread(rng, 64, 7168), "k": 32 * _spread(rng, 4, 512),
                "dtype": rng.choice(["bf16", "fp16"])}
    experts = _spread(rng, 4, 64)
    of = experts * rng.choice([1, 1, 2])
    top = rng.randint(1, min(8, of))
    if op == "experts":
        return {"op": op, "tokens": _spread(rng, 1, 2048), "top": top, "experts": experts, "of": of,
                "k": 32 * _spread(rng, 8, 128), "n": _spread(rng, 128, 2048), "gated": rng.choice([True, False]),
                "dtype": rng.choice(["bf16", "fp16"])}
    hidden = 32 * _spread(rng, 4, 127)
    if op == "dispatch":
        return {"op": op, "tokens": _spread(rng, 1, 4096), "top": min(top, 4), "experts": experts, "of": of,
                "hidden": hidden, "dtype": dtype}
    if op == "train":
        return {"op": op, "tokens": _spread(rng, 1, 4096), "top": min(top, 4), "experts": experts, "of": of,
                "hidden": hidden + rng.choice([0, 0, 1, 6]), "dtype": dtype}
    return {"op": op, "tokens": _spread(rng, 1, 4096), "top": top, "experts": experts, "of": of, "hidden": hidden,
            "dtype": dtype}


# ---------------------------------------------------------------- inputs
def _unblocked_to_blocked(rows):
    """Scale bytes [128 b, 4 j] -> the stored order [b, j, 32, 4, 4]."""
    b, j = rows.shape[0] // 128, rows.shape[1] // 4
    return rows.view(b, 4, 32, j, 4).permute(0, 3, 2, 1, 4).contiguous()


def _power(e):
    """float32 2^e of whole e in [-126, 127], exact (pow is not)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x):
    """Packed codes [rows, K/2] and scale bytes [rows, K/32] of x [rows, K] (inputs of the products)."""
    rows, k = x.shape
    blocks = x.float().view(rows, k // 32, 32)
    exponent = torch.frexp(blocks.abs().amax(-1)).exponent - 3
    v = (blocks * _power(-exponent).unsqueeze(-1)).abs()
    code = torch.bucketize(v, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device))
    code = (code + 8 * (blocks < 0)).to(torch.uint8).view(rows, k // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), (exponent + 127).to(torch.uint8)


def _operand(gen, rows, k, std):
    """A quantised operand: packed [rows, K/2], scales in the stored order, rows and columns padded."""
    packed, sc = _encode(torch.randn((rows, k), generator=gen, device="cuda") * std)
    full = torch.zeros((-(-rows // 128) * 128, -(-k // 128) * 4), dtype=torch.uint8, device="cuda")
    full[:rows, :k // 32] = sc
    return packed, _unblocked_to_blocked(full)


def _routes(gen, case):
    """Each token's experts [T, top] and weights; some experts are in more demand than others."""
    logits = torch.randn((case["tokens"], case["of"]), generator=gen, device="cuda")
    logits += 0.5 * torch.randn((case["of"],), generator=gen, device="cuda")
    top, ids = torch.topk(logits, case["top"], dim=1)
    return ids, torch.softmax(top, 1)


def _sorted(ids, experts):
    """order, slots and offsets of slots sorted by expert."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    counts = (key.unsqueeze(1) == torch.arange(experts, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    slots = torch.where(key < experts, place, -1).view_as(ids)
    routed = torch.arange(order.numel(), device=order.device) < offsets[-1]
    order = torch.where(routed, order, -1)
    return order.to(torch.int32), slots.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if op == "quantize":
        # activations: a few channels are much larger than the others
        x = randn(case["rows"], case["cols"]) * torch.exp(randn(case["cols"]))
        return {"case": case, "x": x.to(dtype)}
    if op == "gemm":
        return {"case": case, "a": _operand(gen, case["m"], case["k"], 1.0),
                "b": _operand(gen, case["n"], case["k"], case["k"] ** -0.5)}
    ids, weights = _routes(gen, case)
    state = {"case": case, "ids": ids, "weights": weights}
    tokens, experts = case["tokens"], case["experts"]
    if op == "dispatch":
        state["x"] = randn(tokens, case["hidden"]).to(dtype)
        return state
    rows = tokens * case["top"]
    order, slots, offsets = _sorted(ids, experts)
    state |= {"order": order, "slots": slots, "offsets": offsets}
    if op == "experts":
        k, n = case["k"], case["n"]
        counts = (offsets[1:] - offsets[:-1]).tolist()
        state["capacity"] = max(1, max(counts))  # for the plain form's padded batch
        packed, sc = _encode(randn(rows, k))
        # scales: each expert's rows begin a block of 128
        full = torch.zeros(((min(rows, experts) + rows // 128) * 128, -(-k // 128) * 4), dtype=torch.uint8,
                           device="cuda")
        full[:, :k // 32][_scale_rows(offsets, rows)] = sc
        state["a"] = (packed, _unblocked_to_blocked(full))
        state["b"] = [tuple(torch.stack(t) for t in zip(*(_operand(gen, n, k, k ** -0.5) for _ in range(experts))))
                      for _ in range(2 if case["gated"] else 1)]
        return state
    state["ys"] = randn(rows, case["hidden"]).to(dtype)
    if op == "train":
        state["x"] = randn(tokens, case["hidden"]).to(dtype)
        state["dy"] = randn(tokens, case["hidden"]).to(dtype)
        state["dxs"] = randn(rows, case["hidden"]).to(dtype)
    return state


# ---------------------------------------------------------------- plain forms
def _scale_rows(offsets, rows):
    """The row of each sorted row's scales: every expert begins at a multiple of 128 (rows behind the last
    expert's get the last row that is there)."""
    offsets = offsets.long()
    blocks = (offsets[1:] - offsets[:-1] + 127) // 128
    first = torch.cat([blocks.new_zeros(1), blocks.cumsum(0)]) * 128
    r = torch.arange(rows, device=offsets.device)
    e = (r.unsqueeze(1) >= offsets[1:]).sum(1)
    last = offsets.numel() - 1
    inside = first[e.clamp(max=last - 1)] + r - offsets[e.clamp(max=last - 1)]
    return torch.where(e < last, inside, torch.full_like(inside, (min(rows, last) + rows // 128) * 128 - 1))


def _decode(packed, scales, where=None):
    """float32 values [rows, K] of packed codes and scales in the stored order (`where`: the scales' rows)."""
    b, j = scales.shape[0], scales.shape[1]
    sc = scales.permute(0, 3, 2, 1, 4).reshape(b * 128, j * 4)
    rows, k = packed.shape[0], packed.shape[1] * 2
    sc = (sc[:rows] if where is None else sc[where])[:, :k // 32]
    codes = torch.stack([packed & 15, packed >> 4], -1).view(rows, k // 32, 32)
    m = (codes & 7).float()
    v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, m * 2 - 8))
    v = torch.where(codes > 7, -v, v)
    half = sc.to(torch.int32) - 127
    lower = torch.div(half, 2, rounding_mode="floor")
    return (v * _power(lower).unsqueeze(-1) * _power(half - lower).unsqueeze(-1)).view(rows, k)


def _round_to_mxfp4(x):
    """The values that x [rows, K] has as MXFP4 (K % 32 == 0)."""
    blocks = x.float().view(x.shape[0], x.shape[1] // 32, 32)
    amax = blocks.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(min=-127)
    v = blocks * _power(-e)
    m = v.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = (torch.round(m / step) * step).clamp(max=6.0)
    lower = torch.div(e, 2, rounding_mode="floor")  # 2^-127 is not a normal number
    return (torch.where(v < 0, -m, m) * _power(lower) * _power(e - lower)).view_as(x)


def _plain(s):
    case = s["case"]
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    if op == "quantize":
        x = s["x"]
        if case["axis"] == 0:
            x = torch.nn.functional.pad(x, (0, 0, 0, -x.shape[0] % 32)).t().contiguous()
        return _round_to_mxfp4(x).to(torch.bfloat16)
    if op == "gemm":
        return (_decode(*s["a"]) @ _decode(*s["b"]).t()).to(dtype)
    if op == "experts":
        offsets, experts, cap = s["offsets"].long(), case["experts"], s["capacity"]
        a = _decode(*s["a"], _scale_rows(s["offsets"], s["a"][0].shape[0]))
        rows = offsets[:-1, None] + torch.arange(cap, device=a.device)  # [E, cap]
        padded = a[rows.clamp(max=a.shape[0] - 1)]
        ys = []
        for packed, scales in s["b"]:
            w = _decode(packed.flatten(0, 1), scales.flatten(0, 1), _weight_rows(packed))
            ys.append(torch.bmm(padded, w.view(experts, case["n"], case["k"]).transpose(1, 2)))
        y = ys[0] * torch.sigmoid(ys[0]) * ys[1] if case["gated"] else ys[0]
        r = torch.arange(a.shape[0], device=a.device)
        e = (r.unsqueeze(1) >= offsets[1:]).sum(1)
        here = e < experts
        e = e.clamp(max=experts - 1)
        y = y[e, (r - offsets[e]).clamp(max=cap - 1)]
        return torch.where(here.unsqueeze(1), y, 0.0).to(dtype)
    if op == "dispatch":
        order, slots, offsets = _sorted(s["ids"], case["experts"])
        values = _round_to_mxfp4(s["x"])[(order // case["top"]).clamp(min=0)]
        return order, slots, offsets, torch.where(order.unsqueeze(1) >= 0, values, 0.0).to(torch.bfloat16)
    here = (s["slots"] >= 0).unsqueeze(-1)
    taken = torch.where(here, s["ys"][s["slots"].clamp(min=0)].float(), 0.0)  # [T, top, H]
    y = (s["weights"].unsqueeze(-1) * taken).sum(1).to(dtype)
    if op == "combine":
        return y
    routed = (s["order"] >= 0).unsqueeze(1)
    order = s["order"].clamp(min=0)
    token = order // case["top"]
    xs = torch.where(routed, s["x"][token], 0)
    dx = torch.where(here, s["dxs"][s["slots"].clamp(min=0)].float(), 0.0).sum(1).to(dtype)
    dy = s["dy"].float()
    dys = torch.where(routed, s["weights"].view(-1)[order].unsqueeze(1) * dy[token], 0.0).to(dtype)
    dw = (taken * dy.unsqueeze(1)).sum(-1)
    return xs, dx, y, dys, dw


def _weight_rows(packed):
    """Rows of the scales of stacked weights [E, N, K/2]: each expert's begin at a multiple of 128."""
    e, n = packed.shape[0], packed.shape[1]
    padded = -(-n // 128) * 128
    return (torch.arange(e, device=packed.device)[:, None] * padded + torch.arange(n, device=packed.device)).view(-1)


# ---------------------------------------------------------------- the framework's operators
_modules = None


def _framework():
    global _modules
    if _modules is None:
        sys.path.insert(0, os.path.abspath("reference-kernels_b200"))
        from nvfp4_b200 import moe, mx
        _modules = mx, moe
    return _modules


def _own(s):
    mx, moe = _framework()
    case = s["case"]
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    if op == "quantize":
        return mx.dequantize(*mx.quantize(s["x"], axis=case["axis"]), dtype=torch.bfloat16)
    if op == "gemm":
        return mx.gemm(*s["a"], *s["b"], out_dtype=dtype)
    if op == "experts":
        if case["gated"]:
            return mx.dual_gemm(*s["a"], *s["b"][0], *s["b"][1], offsets=s["offsets"], out_dtype=dtype)
        return mx.gemm(*s["a"], *s["b"][0], offsets=s["offsets"], out_dtype=dtype)
    if op == "dispatch":
        routing = moe.sort(s["ids"], case["experts"])
        packed, scales = moe.quantize_tokens(s["x"], routing)
        return (routing.order, routing.slots, routing.offsets,
                mx.dequantize(packed, scales, offsets=routing.offsets, dtype=torch.bfloat16))
    routing = moe.Routing(s["order"], s["slots"], s["offsets"])
    y = moe.combine(s["ys"], s["weights"], routing)
    if op == "combine":
        return y
    dys, dw = moe.combine_backward(s["dy"], s["ys"], s["weights"], routing)
    return moe.gather(s["x"], routing), moe.gather_backward(s["dxs"], routing), y, dys, dw


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- cost
def _code_bytes(rows, k):
    return rows * (k // 2 + k // 32)


def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        # x once, the codes and scales once written and once read, the values once (2 bytes)
        return {"bytes": n * size + 2 * (n / 2 + n / 32) + 2 * n, "flops": 0}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _code_bytes(m + n, k) + m * n * size, "flops": 2 * m * n * k}
    tokens, top, experts = case["tokens"], case["top"], case["experts"]
    rows = tokens * top * experts / case["of"]  # routed here, on average
    if op == "experts":
        busy = experts * (1 - (1 - 1 / experts) ** rows)  # experts with a token, on average
        products = 2 if case["gated"] else 1
        return {"bytes": rows * case["k"] * (1 / 2 + 1 / 32) + products * busy * _code_bytes(case["n"], case["k"])
                + tokens * top * case["n"] * size,
                "flops": 2 * products * rows * case["n"] * case["k"]}
    hidden = case["hidden"]
    if op == "dispatch":
        # ids, x, three lists, the routed rows' codes written and read, all rows' values
        return {"bytes": tokens * top * 16 + tokens * hidden * size + 2 * rows * hidden * (1 / 2 + 1 / 32)
                + tokens * top * hidden * 2, "flops": 0}
    combine = tokens * top * 8 + rows * hidden * size + tokens * hidden * size
    if op == "combine":
        return {"bytes": combine, "flops": 2 * rows * hidden}
    # x, dy and y by token; ys, dxs, xs and dys by row
    return {"bytes": combine + tokens * hidden * size * 3 + (rows + 2 * tokens * top) * hidden * size,
            "flops": 7 * rows * hidden}


# ---------------------------------------------------------------- the definition, in 64 bits
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _values64(packed, scale_bytes):
    """float64 [rows, K] of packed [rows, K/2] and plain scale bytes [rows, K/32]."""
    table = torch.tensor(_E2M1, dtype=torch.float64, device=packed.device)
    v = torch.empty((packed.shape[0], packed.shape[1] * 2), dtype=torch.float64, device=packed.device)
    v[:, 0::2] = table[(packed % 16).long()]
    v[:, 1::2] = table[(packed // 16).long()]
    return v * _power64(scale_bytes.long() - 127).repeat_interleave(32, dim=1)


def _scales64(scales, first, rows, k):
    """Plain scale bytes [rows, K/32] of the rows from block `first` on, by the stored order's own address rule:
    byte (i, j) of a block of 128 rows and 4 columns is at (i % 32) * 16 + (i // 32) * 4 + j."""
    blocks_k = scales.shape[1]
    i = torch.arange(rows, device=scales.device)[:, None]
    j = torch.arange(k // 32, device=scales.device)[None, :]
    at = ((first + i // 128) * blocks_k + j // 4) * 512 + (i % 32) * 16 + (i % 128) // 32 * 4 + j % 4
    return scales.reshape(-1)[at]


def _mxfp4_64(x):
    """MXFP4 values of float64 x [rows, K] by the nearest of the 8 magnitudes, ties to the even code."""
    b = x.reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    powers = _power64(torch.arange(-149, 129, device=x.device))
    floor = torch.searchsorted(powers, amax, right=True) - 150  # floor(log2(amax))
    s = _power64((floor - 2).clamp(-127, 127))
    m = (b / s).abs()
    out = torch.zeros_like(m)
    grid = _E2M1[:8]
    for code in range(1, 8):
        half = (grid[code - 1] + grid[code]) / 2
        out = torch.where((m > half) | ((m == half) & (code % 2 == 0)), grid[code], out)
    return (out * torch.sign(b) * s).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].double()
        if case["axis"] == 0:
            full = torch.zeros((-(-x.shape[0] // 32) * 32, x.shape[1]), dtype=torch.float64, device=x.device)
            full[:x.shape[0]] = x
            x = full.t()
        return torch.cat([_mxfp4_64(part) for part in x.split(1024)])
    if op == "gemm":
        k = case["k"]
        a = _values64(s["a"][0], _scales64(s["a"][1], 0, case["m"], k))
        b = _values64(s["b"][0], _scales64(s["b"][1], 0, case["n"], k))
        return a @ b.t()
    top = case["top"]
    if op == "experts":
        k, n = case["k"], case["n"]
        y = torch.zeros((case["tokens"] * top, n), dtype=torch.float64, device="cuda")
        offsets, block = s["offsets"].tolist(), 0
        for e in range(case["experts"]):
            r0, r1 = offsets[e], offsets[e + 1]
            if r0 == r1:
                continue
            a = _values64(s["a"][0][r0:r1], _scales64(s["a"][1], block, r1 - r0, k))
            ys = [a @ _values64(p[e], _scales64(sc[e], 0, n, k)).t() for p, sc in s["b"]]
            y[r0:r1] = ys[0] / (1 + torch.exp(-ys[0])) * ys[1] if case["gated"] else ys[0]
            block += -(-(r1 - r0) // 128)
        return y
    # sorted places, slot by slot on the host
    ids = s["ids"].reshape(-1).tolist()
    lists = [[] for _ in range(case["experts"])]
    for slot, e in enumerate(ids):
        if 0 <= e < case["experts"]:
            lists[e].append(slot)
    order = [slot for one in lists for slot in one]
    routed = torch.tensor(order, dtype=torch.long, device="cuda")
    rows = len(ids)
    if op == "dispatch":
        values = torch.zeros((rows, case["hidden"]), dtype=torch.float64, device="cuda")
        coded = torch.cat([_mxfp4_64(part) for part in s["x"].double().split(1024)])
        values[:len(order)] = coded[routed // top]
        return None, None, None, values
    token, w = routed // top, s["weights"].double().view(-1)
    ys = s["ys"][:len(order)].double()

    def per_token(values):
        out = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda")
        return out.index_add_(0, token, values)

    def per_row(values):
        out = torch.zeros((rows, case["hidden"]), dtype=torch.float64, device="cuda")
        out[:len(order)] = values
        return out

    y = per_token(w[routed, None] * ys)
    if op == "combine":
        return y
    dy = s["dy"].double()
    dw = torch.zeros(rows, dtype=torch.float64, device="cuda")
    dw[routed] = torch.linalg.vecdot(dy[token], ys)
    return (per_row(s["x"].double()[token]), per_token(s["dxs"][:len(order)].double()), y,
            per_row(w[routed, None] * dy[token]), dw.view(case["tokens"], top))
