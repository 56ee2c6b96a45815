"""Plain 64-bit forms of the MXFP4 operators and of the expert routing, for the tests."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], np.float64)


def encode(x):
    """Codes [rows, K] and scale bytes [rows, K/32] of x [rows, K] (K % 32 == 0)."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    amax = np.abs(b).max(-1) if b.size else np.zeros((rows, k // 32))
    # floor(log2(amax)) from the binary exponent: amax = m * 2^e with m in [0.5, 1)
    e = np.where(amax > 0, np.frexp(amax)[1] - 1, -1000) - 2
    e = np.maximum(e, -127)
    q = np.abs(b) / np.ldexp(1.0, e)[..., None]
    # nearest magnitude, ties to the even code, above the largest to the largest
    codes = np.zeros(b.shape, np.int64)
    for c in range(1, 8):
        half = (E2M1[c - 1] + E2M1[c]) / 2
        codes = np.where((q > half) | ((q == half) & (c % 2 == 0)), c, codes)
    codes = codes + 8 * (np.signbit(b) & ~bad[..., None])
    return codes.reshape(rows, k).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def decode(codes, scales):
    """float64 [rows, K] of codes [rows, K] and scale bytes [rows, K/32]."""
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(s, 32, axis=1)


def unpack(packed):
    """uint8 [rows, K/2] -> codes [rows, K]."""
    out = np.empty((packed.shape[0], packed.shape[1] * 2), np.uint8)
    out[:, 0::2] = packed & 15
    out[:, 1::2] = packed >> 4
    return out


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def plain_scales(blocked, rows, k, at=None):
    """Scale bytes [rows, K/32] from the stored order [blocks, K128, 32, 4, 4]; `at`: the rows' scale rows."""
    r = (np.arange(rows) if at is None else np.asarray(at, np.int64))[:, None]
    j = np.arange(k // 32)[None, :]
    return blocked[r // 128, j // 4, r % 32, (r % 128) // 32, j % 4]


def blocked_scales(plain, at=None, blocks=None, fill=0):
    """Scale bytes [rows, K/32] -> the stored order."""
    rows, n = plain.shape
    out = np.full((-(-rows // 128) if blocks is None else blocks, -(-n // 4), 32, 4, 4), fill, np.uint8)
    r = (np.arange(rows) if at is None else np.asarray(at, np.int64))[:, None]
    j = np.arange(n)[None, :]
    out[r // 128, j // 4, r % 32, (r % 128) // 32, j % 4] = plain
    return out


def scale_rows(offsets):
    """The scale row of each row that an expert has, and the number of row blocks in use."""
    at, block = [], 0
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        at.append(block * 128 + np.arange(hi - lo))
        block += -(-(hi - lo) // 128)
    return np.concatenate(at) if at else np.zeros(0, np.int64), block


def route(ids, experts):
    """order, slots, offsets of moe.sort."""
    flat = [int(v) for v in np.asarray(ids).reshape(-1)]
    lists = [[] for _ in range(experts)]
    for s, e in enumerate(flat):
        if 0 <= e < experts:
            lists[e].append(s)
    order = [s for one in lists for s in one]
    slots = np.full(len(flat), -1, np.int64)
    slots[order] = np.arange(len(order))
    offsets = np.concatenate([[0], np.cumsum([len(one) for one in lists])])
    return (np.array(order + [-1] * (len(flat) - len(order)), np.int64), slots.reshape(np.asarray(ids).shape),
            offsets.astype(np.int64))
