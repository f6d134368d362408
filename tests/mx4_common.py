"""Plain 64-bit restatements of microscaled 4-bit rows, their products and the experts' step over them. Nothing here calls a launcher."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDDLES = (LEVELS[1:] + LEVELS[:-1]) / 2
# an f32 step relative to the value: what a sum is off by at most, however the matrix cores round it
STEP = 2.0 ** -23


def row_bytes(k):
    return 16 * -(-k // 32)


def row_scales(k):
    return 16 * -(-k // 512)


def encode(x):
    """(codes, scales) of rows: a byte a code, a byte a block; codes behind the k-th value 0, no padding of the scales. A block that is not finite: 0, 255."""
    x = np.asarray(x, np.float64)
    m, k = x.shape
    blocks = -(-k // 32)
    v = np.zeros((m, 32 * blocks))
    v[:, :k] = x
    v = v.reshape(m, blocks, 32)
    bad = ~np.isfinite(v).all(axis=2)
    v = np.where(bad[:, :, None], 0.0, v)
    most = np.abs(v).max(axis=2)
    e = np.clip(np.where(most > 0, np.frexp(most)[1] - 3, -127), -127, 127)
    size = np.ldexp(np.abs(v), -e[:, :, None])
    codes = (size[..., None] > MIDDLES).sum(axis=3)
    at = np.minimum(codes, 6)
    codes += (codes < 7) & (size == MIDDLES[at]) & (codes % 2 == 1)  # halfway from an odd code: up
    codes |= np.signbit(v) * 8
    return codes.reshape(m, -1).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def pack(codes, scales, k, pad=0):
    """Codes as bytes and scales padded with `pad` bytes, as a device buffer holds them."""
    m = codes.shape[0]
    out = np.full((m, row_scales(k)), pad, np.uint8)
    out[:, :scales.shape[1]] = scales
    return np.ascontiguousarray(codes[:, 0::2] | codes[:, 1::2] << 4), out


def unpack(words, scales, k):
    """(codes, scales) of a device buffer's rows."""
    m = words.shape[0]
    codes = np.zeros((m, 2 * words.shape[1]), np.uint8)
    codes[:, 0::2], codes[:, 1::2] = words & 15, words >> 4
    return codes, scales[:, :-(-k // 32)]


def decode(codes, scales, k):
    v = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    with np.errstate(invalid="ignore"):
        s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v.reshape(v.shape[0], -1, 32) * s[:, :, None]).reshape(v.shape[0], -1)[:, :k]


def some_rows(rng, rows, k, spread=3):
    """Rows of any codes, with scales near 2^-6."""
    blocks = -(-k // 32)
    codes = rng.integers(0, 16, (rows, 32 * blocks)).astype(np.uint8)
    return codes, (121 + rng.integers(-spread, spread + 1, (rows, blocks))).astype(np.uint8)


def product_bound(x, w):
    """x w^T in 64 bits and how far a sum in f32 may be from it: the blocks' sums of products are exact, a step of what they add up to for each of
    them, eight more for the parts that waves add."""
    blocks = -(-x.shape[1] // 32)
    return x @ w.T, (blocks + 8) * STEP * (np.abs(x) @ np.abs(w).T)


def rule_value(g, u):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def moe(x, sel, weights, wg, wu, wd, n_experts, resid, kept):
    """The experts' step in 64 bits, and how far f32 sums may be from it. wg, wu, wd: experts x rows x values. kept: what h and its rule are off by,
    relative. A sum of n values: a step for every 32 of them in each of three parts that a value may be taken in, 64 more for what waves and lanes add."""
    m, top_k = sel.shape
    hidden, ff = x.shape[1], wg.shape[1]

    def steps(n):
        return (3 * -(-n // 32) + 64) * STEP

    y = np.zeros((m, hidden)) if resid is None else resid.astype(np.float64).copy()
    off, size = np.zeros_like(y), np.abs(y)
    for t in range(m):
        for s in range(top_k):
            e = int(sel[t, s])
            if e >= n_experts:
                continue
            g, u = wg[e] @ x[t], wu[e] @ x[t]
            dg, du = steps(hidden) * (np.abs(wg[e]) @ np.abs(x[t])), steps(hidden) * (np.abs(wu[e]) @ np.abs(x[t]))
            h = rule_value(g, u)
            silu = np.abs(rule_value(g, 1.0))
            dh = 1.1 * dg * (np.abs(u) + du) + (silu + 1.1 * dg) * du + kept * np.abs(h)  # silu's slope is below 1.1
            d, w = wd[e] @ h, float(weights[t, s])
            off[t] += abs(w) * (np.abs(wd[e]) @ dh + steps(ff) * (np.abs(wd[e]) @ (np.abs(h) + dh)))
            size[t] += np.abs(w * d)
            y[t] += w * d
    return y, off + (top_k + 1) * STEP * (size + off)
