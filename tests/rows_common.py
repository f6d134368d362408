"""Rows of f32, f16 and bf16 elements on host and device, and plain 64-bit restatements of the 8-bit products and of the rows sorted by
expert and back. Nothing here calls a launcher."""
import numpy as np
import torch

import bloomery_amd as bm

TORCH = {bm.F32: torch.float32, bm.F16: torch.float16, bm.BF16: torch.bfloat16}
NUMPY = {bm.F32: np.float32, bm.F16: np.uint16, bm.BF16: np.uint16}
NAMES = {bm.F32: "f32", bm.F16: "f16", bm.BF16: "bf16"}
# a rounding's largest error relative to the value: half a step
HALF_STEP = {t: torch.finfo(d).eps / 2 for t, d in TORCH.items()}


def rounded(x, dtype):
    """The values of x as elements of dtype, in f64."""
    return torch.from_numpy(np.asarray(x, np.float32)).to(TORCH[dtype]).double().numpy()


def bits(x, dtype):
    """x rounded to elements of dtype, as the words a device buffer holds."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype])
    return t.numpy() if dtype == bm.F32 else t.view(torch.int16).numpy().view(np.uint16)


def values(words, dtype):
    """Device words as f64 values."""
    words = np.ascontiguousarray(words)
    if dtype == bm.F32:
        return words.view(np.float32).astype(np.float64)
    return torch.from_numpy(words.view(np.int16)).view(TORCH[dtype]).double().numpy()


def lines(x, dtype, ld, fill=0.0):
    """A matrix as words with rows ld apart, `fill` between them."""
    x = np.asarray(x, np.float32)
    wide = np.full((x.shape[0], ld), fill, np.float32)
    wide[:, :x.shape[1]] = x
    return bits(wide, dtype)


def codes_of(x):
    """(codes, scales) of f32 rows by the rule: s = f32(amax / 127), the quotients in f64 (a quotient of two f32 numbers next to a half is
    further from it than f64's rounding, or on it)."""
    x = np.asarray(x, np.float32)
    amax = np.abs(x).max(axis=1)
    bad = ~np.isfinite(x).all(axis=1)
    with np.errstate(all="ignore"):
        s = (amax / np.float32(127.0)).astype(np.float32)
        q = np.clip(np.rint(x.astype(np.float64) / s.astype(np.float64)[:, None]), -127, 127)
    q[(s == 0) | bad] = 0
    s[bad] = np.nan
    return q.astype(np.int8), s


def product(q, s, w, ws):
    """The product's value before its last rounding, with the f32 roundings of the rule: bit for bit what the kernels form."""
    sums = q.astype(np.int64) @ w.astype(np.int64).T
    with np.errstate(over="ignore", invalid="ignore"):
        return (sums.astype(np.float32) * s[:, None]).astype(np.float32) * ws[None, :].astype(np.float32)


def padded(codes, k):
    out = np.zeros((codes.shape[0], -(-k // 16) * 16), np.int8)
    out[:, :k] = codes
    return out


def tables(ids, n_experts):
    """order, start, place of flat ids (unlisted: 0xffffffff)."""
    ids = np.asarray(ids, np.uint32).reshape(-1)
    order = [s for e in range(n_experts) for s in np.flatnonzero(ids == e)]
    start = np.concatenate([[0], np.cumsum([np.count_nonzero(ids == e) for e in range(n_experts)])])
    place = np.full(ids.size, 0xFFFFFFFF, np.uint32)
    place[order] = np.arange(len(order), dtype=np.uint32)
    return np.array(order, np.uint32), start.astype(np.uint32), place
