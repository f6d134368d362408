"""GPU tests of microscaled 4-bit floating point (bm_mx4_*) against plain numpy in 64 bits: codes, scales and the values that they stand for
exactly; products and the experts' step within the f32 steps of their sums and one rounding to the output's type."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
import mx4_common as mx
from common import normal_f32
from rows_common import HALF_STEP, NAMES, NUMPY, TORCH, bits, lines, rounded, tables, values

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)


@pytest.fixture(scope="module")
def gpu():
    g = bm.Gpu(0)
    yield g
    g.close()


class Held:
    """Device buffers of a test, freed at its end."""

    def __init__(self, gpu):
        self.gpu, self.all = gpu, []

    def up(self, host):
        return self.keep(self.gpu.upload(np.ascontiguousarray(host)))

    def out(self, dtype, count, byte=0xEE):
        return self.keep(self.gpu.buffer(dtype, count).fill_bytes(byte))

    def keep(self, b):
        self.all.append(b)
        return b

    def free(self):
        for b in self.all:
            b.free()


@pytest.fixture
def held(gpu):
    h = Held(gpu)
    yield h
    h.free()


def clean(gpu):
    assert gpu.fault() == (bm.FAULT_NONE, 0)


def quantize(gpu, held, x, dtype, ld=None, live=None):
    m, k = x.shape
    xd = held.up(lines(x, dtype, ld or k, np.nan))
    codes, scales = held.out(np.uint8, m * mx.row_bytes(k), 0x55), held.out(np.uint8, m * mx.row_scales(k), 0x55)
    gpu.enqueue_mx4_quantize(xd, dtype, m, k, codes, scales, ld_x=ld, live=live)
    return codes, scales


def assert_rows(codes, scales, x):
    m, k = x.shape
    words, padded = mx.pack(*mx.encode(x), k)
    assert np.array_equal(scales.download().reshape(m, -1), padded)
    assert np.array_equal(codes.download().reshape(m, -1), words)


def up_rows(held, codes, scales, k, junk=None):
    """Rows on the device; junk: what stands behind the last block's scale, and in codes behind the k-th value."""
    if junk is not None:
        codes = codes.copy()
        codes[:, k:] = junk & 15
    words, padded = mx.pack(codes, scales, k, junk or 0)
    return held.up(words), held.up(padded)


def zeroed(codes, k):
    codes = codes.copy()
    codes[:, k:] = 0
    return codes


def assert_near(words, dtype, exact, bound):
    got = values(words, dtype).reshape(exact.shape)
    off = HALF_STEP[dtype] * (np.abs(exact) + bound) + bound
    if dtype == bm.F16:
        off += 2.0 ** -25  # half of the smallest step
    worst = np.max(np.abs(got - exact) - off)
    assert np.isfinite(got).all() and worst <= 0, worst


# ------------------------------------------------------------------------------------------------ quantizer

SIZES = ((1, 1, 1), (5, 2, 3), (7, 15, 15), (6, 31, 33), (9, 32, 32), (5, 33, 33), (5, 500, 500), (5, 512, 515), (3, 513, 513), (4, 1024, 1024),
         (3, 1996, 1997), (5, 2048, 2048), (2, 5000, 5001), (2, 8200, 8200), (1, 131072, 131072), (257, 64, 64), (3000, 40, 40))


@DTYPES
@pytest.mark.parametrize("m,k,ld", SIZES)
def test_codes_are_the_rules_and_come_back(gpu, held, dtype, m, k, ld):
    rng = np.random.default_rng(100 + m + k)
    x = rounded(normal_f32(rng, (m, k)) * np.exp(2 * normal_f32(rng, (m, 1))), dtype)
    codes, scales = quantize(gpu, held, x, dtype, ld)
    assert_rows(codes, scales, x)
    y = held.out(NUMPY[dtype], m * ld)
    gpu.enqueue_mx4_dequantize(codes, scales, m, k, y, dtype, ld_y=ld)
    got = y.download().reshape(m, ld)
    assert np.array_equal(got[:, :k], bits(mx.decode(*mx.encode(x), k), dtype))
    assert (got[:, k:].view(np.uint8) == 0xEE).all()
    clean(gpu)


def test_every_scale_its_halves_and_their_neighbours(gpu, held):
    """Blocks whose largest value lies anywhere in f32, holding the values halfway between codes and their f32 neighbours."""
    half = np.array([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    rows = []
    for e in range(-149, 126):
        for top in (4.0, 6.0, 7.9999995):
            v = np.concatenate([half, np.nextafter(half, np.float32(9)), np.nextafter(half, np.float32(-9)), [0.5, 1, 1.5, 2, 3, top, 6.5 if top > 6.5 else 1, -0.0]])
            v = v.astype(np.float64) * rng_signs(len(v))
            with np.errstate(over="ignore"):
                v = np.ldexp(v, e).astype(np.float32)
            rows.append(np.where(np.isfinite(v), v, np.float32(1)))
    x = np.stack(rows)
    codes, scales = quantize(gpu, held, x, bm.F32)
    assert_rows(codes, scales, x)
    clean(gpu)


def rng_signs(n):
    return np.where(np.arange(n) * 7 % 3 == 0, -1.0, 1.0)


@DTYPES
def test_every_code_under_every_scale_comes_back(gpu, held, dtype):
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    c, s = up_rows(held, codes, scales, 32)
    y = held.out(NUMPY[dtype], 256 * 32)
    gpu.enqueue_mx4_dequantize(c, s, 256, 32, y, dtype)
    got = values(y.download(), dtype).reshape(256, 32)
    with np.errstate(over="ignore"):
        want = values(bits(mx.decode(codes, scales, 32), dtype), dtype).reshape(256, 32)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[255]).all()
    assert np.array_equal(got[:255], want[:255])


@pytest.mark.parametrize("k", (40, 700, 2000, 9000))
@pytest.mark.parametrize("value", (np.nan, np.inf, -np.inf))
def test_a_block_that_is_not_finite(gpu, held, k, value):
    rng = np.random.default_rng(7)
    x = normal_f32(rng, (4, k))
    x[1, k - 1] = value
    gpu.fault_clear()
    codes, scales = quantize(gpu, held, x, bm.F32)
    assert_rows(codes, scales, x)
    assert gpu.fault()[0] & 0xFF == bm.SITE_QUANT_COLUMN
    gpu.fault_clear()


@pytest.mark.parametrize("k", (48, 2048, 9000))
def test_rows_behind_the_live_ones_keep_what_they_held(gpu, held, k):
    rng = np.random.default_rng(8)
    x = normal_f32(rng, (6, k))
    words, padded = mx.pack(*mx.encode(x), k)
    for live in (0, 1, 4, 6, 1000):
        codes, scales = quantize(gpu, held, x, bm.F32, live=held.up(np.array([live], np.uint32)))
        c, s = codes.download().reshape(6, -1), scales.download().reshape(6, -1)
        n = min(live, 6)
        assert np.array_equal(c[:n], words[:n]) and np.array_equal(s[:n], padded[:n])
        assert (c[n:] == 0x55).all() and (s[n:] == 0x55).all()
    clean(gpu)


RULES = ((None, lambda g, u: g / (1 + np.exp(-g)) * u),
         ((bm.ACT_SWIGLU_CLAMP, 1.5), lambda g, u: np.minimum(g / (1 + np.exp(-g)), 1.5) * np.clip(u, -1.5, 1.5)),
         ((bm.ACT_SWIGLU_OAI, 1.25), lambda g, u: np.minimum(g, 1.25) / (1 + np.exp(-1.702 * np.minimum(g, 1.25))) * (np.clip(u, -1.25, 1.25) + 1)),
         ((bm.ACT_SITU, 2.0), lambda g, u: 2.0 * np.tanh(g / 2.0) / (1 + np.exp(-g)) * 25 * np.tanh(u / 25)),
         ((bm.ACT_SWIGLU_GCLAMP, 1.5), lambda g, u: np.minimum(g, 1.5) / (1 + np.exp(-np.minimum(g, 1.5))) * np.clip(u, -1.5, 1.5)))


@DTYPES
@pytest.mark.parametrize("rule", range(len(RULES)))
@pytest.mark.parametrize("m,k,ld", ((3, 96, 96), (5, 1000, 1003), (40, 2048, 2048)))
def test_codes_behind_a_gate_rule(gpu, held, dtype, rule, m, k, ld):
    """A value is off by 2^-18 of its magnitude at most (of the factors' where a clamp or a tanh cuts): its code is that of a value as near."""
    rng = np.random.default_rng(9 + rule)
    g, u = (rounded(2 * normal_f32(rng, (m, k)), dtype) for _ in range(2))
    codes, scales = held.out(np.uint8, m * mx.row_bytes(k), 0x55), held.out(np.uint8, m * mx.row_scales(k), 0x55)
    gpu.enqueue_mx4_swiglu_quantize(held.up(lines(g, dtype, ld, np.nan)), held.up(lines(u, dtype, ld, np.nan)), dtype, m, k, codes, scales, ld=ld,
                                    rule=RULES[rule][0])
    clean(gpu)
    want = RULES[rule][1](g, u)
    low, high = np.sort(np.stack([want * (1 - 2.0 ** -18), want * (1 + 2.0 ** -18)]), axis=0)
    got_codes, got_scales = mx.unpack(codes.download().reshape(m, -1), scales.download().reshape(m, -1), k)
    got = mx.decode(got_codes, got_scales, k)
    # under the block's scale the value's code, or that of a value as near (the scale too may be that of a largest value as near)
    pad = np.zeros((m, 32 * got_scales.shape[1] - k))
    s = np.ldexp(1.0, got_scales.astype(int) - 127).repeat(32, axis=1)[:, :k]
    for block_of in (low, high):
        most = np.abs(np.concatenate([block_of, pad], 1)).reshape(m, -1, 32).max(axis=2).repeat(32, axis=1)[:, :k]
        assert (most < 8 * s * (1 + 2.0 ** -17)).all() and ((most >= 4 * s * (1 - 2.0 ** -17)) | (s == 2.0 ** -127)).all()

    def code_value(v):
        size = np.abs(v) / s
        n = (size[..., None] > mx.MIDDLES).sum(axis=2)
        n += (n < 7) & (size == mx.MIDDLES[np.minimum(n, 6)]) & (n % 2 == 1)
        return np.sign(v) * mx.LEVELS[n] * s

    assert ((got >= code_value(low)) & (got <= code_value(high))).all()
    assert (got_codes[:, k:] == 0).all()


def test_a_clamped_rule_raises_where_a_sum_is_not_finite(gpu, held):
    g, u = np.ones((2, 64), np.float32), np.ones((2, 64), np.float32)
    g[1, 40] = np.inf
    gpu.fault_clear()
    codes, scales = held.out(np.uint8, 2 * 32), held.out(np.uint8, 2 * 16)
    gpu.enqueue_mx4_swiglu_quantize(held.up(g), held.up(u), bm.F32, 2, 64, codes, scales, rule=(bm.ACT_SWIGLU_CLAMP, 1.0))
    got = scales.download().reshape(2, 16)
    assert got[1, 1] == 255 and got[0, 0] == got[0, 1] == got[1, 0] != 255
    assert gpu.fault()[0] & 0xFF in (bm.SITE_QUANT_COLUMN, bm.SITE_F32_PRODUCT)
    gpu.fault_clear()


# -------------------------------------------------------------------------------------------------- product

PRODUCTS = ((1, 1, 1), (1, 16, 32), (2, 17, 33), (1, 768, 2048), (3, 100, 130), (16, 16, 128), (17, 33, 255), (24, 300, 512), (5, 2000, 96), (33, 64, 1996),
            (64, 48, 513), (100, 129, 700), (130, 260, 1024), (300, 200, 2048), (777, 500, 500), (260, 1000, 160))


@DTYPES
@pytest.mark.parametrize("m,rows,k", PRODUCTS)
def test_product_of_codes(gpu, held, dtype, m, rows, k):
    rng = np.random.default_rng(200 + m + rows + k)
    w, q = some_rows_zeroed(rng, rows, k), some_rows_zeroed(rng, m, k)
    wd, qd = up_rows(held, *w, k, junk=0xFF), up_rows(held, *q, k)
    ld = rows + 3
    y = held.out(NUMPY[dtype], m * ld)
    gpu.enqueue_mx4_gemm(*wd, rows, k, *qd, m, y, dtype, ld_y=ld)
    got = y.download().reshape(m, ld)
    assert_near(got[:, :rows], dtype, *mx.product_bound(mx.decode(*q, k), mx.decode(*w, k)))
    assert (got[:, rows:].view(np.uint8) == 0xEE).all()
    clean(gpu)


def some_rows_zeroed(rng, rows, k):
    codes, scales = mx.some_rows(rng, rows, k)
    return zeroed(codes, k), scales


@pytest.mark.parametrize("m,rows,k", ((1, 40, 64), (8, 100, 1000), (40, 200, 640), (200, 300, 2048)))
def test_scales_far_apart(gpu, held, m, rows, k):
    """Blocks at either end of the scales' range whose products lie in the middle of f32's."""
    rng = np.random.default_rng(3)
    w, q = some_rows_zeroed(rng, rows, k), some_rows_zeroed(rng, m, k)
    middle = rng.integers(4, 251, w[1].shape[1])
    ws = (middle[None, :] + rng.integers(-3, 4, w[1].shape)).astype(np.uint8)
    qs = (254 - middle[None, :] + rng.integers(-3, 4, q[1].shape)).astype(np.uint8)
    y = held.out(np.float32, m * rows)
    gpu.enqueue_mx4_gemm(*up_rows(held, w[0], ws, k), rows, k, *up_rows(held, q[0], qs, k), m, y, bm.F32)
    x, v = mx.decode(q[0], qs, k), mx.decode(w[0], ws, k)
    assert_near(y.download().reshape(m, rows), bm.F32, *mx.product_bound(x, v))
    clean(gpu)


@pytest.mark.parametrize("m,rows,k", ((1, 40, 64), (30, 100, 1000), (300, 400, 640)))
def test_a_nan_scale_is_its_rows_and_its_columns(gpu, held, m, rows, k):
    rng = np.random.default_rng(4)
    w, q = some_rows_zeroed(rng, rows, k), some_rows_zeroed(rng, m, k)
    w[1][rows // 2, -1] = 255
    q[1][m - 1, 0] = 255
    y = held.out(np.float32, m * rows)
    gpu.enqueue_mx4_gemm(*up_rows(held, *w, k), rows, k, *up_rows(held, *q, k), m, y, bm.F32)
    got = y.download().reshape(m, rows)
    want = np.zeros((m, rows), bool)
    want[:, rows // 2] = want[m - 1, :] = True
    assert np.array_equal(np.isnan(got), want)


@DTYPES
@pytest.mark.parametrize("m,rows,k", ((1, 768, 2048), (1, 5, 1), (2, 33, 70), (3, 100, 512), (4, 50, 1996), (7, 300, 2048), (8, 64, 4100), (9, 64, 300), (1, 40, 20000),
                                      (40, 200, 640)))
def test_product_from_rows(gpu, held, dtype, m, rows, k):
    rng = np.random.default_rng(400 + m + rows)
    x = rounded(normal_f32(rng, (m, k)) * np.exp(normal_f32(rng, (m, 1))), dtype)
    w = some_rows_zeroed(rng, rows, k)
    codes, scales = held.out(np.uint8, m * mx.row_bytes(k), 0x55), held.out(np.uint8, m * mx.row_scales(k), 0x55)
    y, ld = held.out(NUMPY[dtype], m * rows), k + 5
    gpu.enqueue_mx4_gemm_x(*up_rows(held, *w, k, junk=0xFF), rows, k, held.up(lines(x, dtype, ld, np.nan)), dtype, m, codes, scales, y, dtype, ld_x=ld)
    assert_rows(codes, scales, x)
    assert_near(y.download().reshape(m, rows), dtype, *mx.product_bound(mx.decode(*mx.encode(x), k), mx.decode(*w, k)))
    clean(gpu)


def picks(rng, m, n, top_k, away=0.0):
    ids = np.argsort(rng.random((m, max(n, top_k))), axis=1)[:, :top_k].astype(np.uint32) % n
    ids[rng.random(ids.shape) < away] = bm.HOST_SLOT
    return ids


@DTYPES
@pytest.mark.parametrize("m,n,top_k,rows,k", ((1, 4, 2, 16, 16), (1, 1, 1, 5, 40), (3, 8, 8, 33, 130), (16, 64, 8, 200, 256), (5, 300, 4, 20, 64),
                                              (40, 6, 3, 257, 320), (200, 5, 2, 130, 192), (150, 3, 3, 300, 1000), (700, 4, 2, 256, 512)))
def test_experts_product_over_shared_and_own_columns(gpu, held, dtype, m, n, top_k, rows, k):
    rng = np.random.default_rng(2000 + m + rows)
    ids = picks(rng, m, n, top_k, 0.1)
    if n > 4:
        ids[ids == 2] = bm.HOST_SLOT  # an expert that nobody picked
    order, start, _ = tables(ids, n)
    n_slots, listed = m * top_k, int(start[-1])
    w = some_rows_zeroed(rng, n * rows, k)
    full = np.full(n_slots, 0x12345678, np.uint32)  # behind the listed entries: what no launch may follow
    full[:listed] = order
    wd, od, sd = up_rows(held, *w, k, junk=0xFF), held.up(full), held.up(start)
    expert, wv = np.repeat(np.arange(n), np.diff(start.astype(np.int64))), mx.decode(*w, k).reshape(n, rows, k)
    for own in (False, True):
        q = some_rows_zeroed(rng, n_slots if own else m, k)
        qd, x = up_rows(held, *q, k), mx.decode(*q, k)
        col = np.arange(listed) if own else order // top_k
        ld = rows + 1
        y = held.out(NUMPY[dtype], n_slots * ld)
        gpu.enqueue_mx4_gemm_experts(*wd, n, rows, k, *qd, None if own else od, sd, n_slots, 0 if own else top_k, y, dtype, ld_y=ld)
        got = y.download().reshape(n_slots, ld)
        for e in range(n):
            at = np.flatnonzero(expert == e)
            if at.size:
                assert_near(got[at, :rows], dtype, *mx.product_bound(x[col[at]], wv[e]))
        assert (got[listed:].view(np.uint8) == 0xEE).all() and (got[:, rows:].view(np.uint8) == 0xEE).all()
    clean(gpu)


@pytest.mark.parametrize("rows", (48, 300))
def test_tables_that_are_none_are_skipped(gpu, held, rows):
    """Runs that run backwards or past the slots, entries that name no slot: raised, nothing out of range read or written."""
    rng = np.random.default_rng(13)
    n, k, n_slots, top_k = 4, 64, 12, 2
    w, q = some_rows_zeroed(rng, n * rows, k), some_rows_zeroed(rng, 6, k)
    wd, qd = up_rows(held, *w, k), up_rows(held, *q, k)
    order = np.arange(12, dtype=np.uint32)
    x, wv = mx.decode(*q, k), mx.decode(*w, k).reshape(n, rows, k)
    for start, ok in (((0, 3, 2, 5, 12), None), ((0, 3, 6, 9, 13), {0: (0, 3), 1: (3, 6), 2: (6, 9)}), ((0, 3, 0xFFFFFFF0, 9, 12), {0: (0, 3), 3: (9, 12)})):
        gpu.fault_clear()
        y = held.out(np.float32, n_slots * rows)
        gpu.enqueue_mx4_gemm_experts(*wd, n, rows, k, *qd, held.up(order), held.up(np.array(start, np.uint32)), n_slots, top_k, y, bm.F32)
        got = y.download().reshape(n_slots, rows)
        if ok:
            done = np.zeros(n_slots, bool)
            for e, (a, b) in ok.items():
                assert_near(got[a:b], bm.F32, *mx.product_bound(x[order[a:b] // top_k], wv[e]))
                done[a:b] = True
            assert (got[~done].view(np.uint32) == 0xEEEEEEEE).all()
        assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    bad = order.copy()
    bad[[1, 7]] = [12, 0xFFFFFFFF]
    gpu.fault_clear()
    y = held.out(np.float32, n_slots * rows)
    gpu.enqueue_mx4_gemm_experts(*wd, n, rows, k, *qd, held.up(bad), held.up(np.array((0, 3, 6, 9, 12), np.uint32)), n_slots, top_k, y, bm.F32)
    got = y.download().reshape(n_slots, rows)
    assert np.isnan(got[[1, 7]]).all() and np.isfinite(np.delete(got, [1, 7], 0)).all()
    assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    gpu.fault_clear()


# ------------------------------------------------------------------------------------ a few tokens' experts

# h and its rule: the rule's f32 operations, and what h is held in: f32's 24 bits, f16 rows' two parts of 8 and 8 (the first cut, the second rounded: off by
# 2^-9 of what is below 2^-7), bf16 rows' one rounding, half a step
KEPT = {bm.F32: 2.0 ** -20, bm.F16: 2.0 ** -15, bm.BF16: 2.0 ** -20 + HALF_STEP[bm.BF16]}


class Stack:
    def __init__(self, held, rng, n, hidden, ff, junk=0xFF):
        self.n, self.hidden, self.ff = n, hidden, ff
        self.dev, self.host = {}, {}
        for name, rows, k in (("gate", ff, hidden), ("up", ff, hidden), ("down", hidden, ff)):
            w = some_rows_zeroed(rng, n * rows, k)
            self.dev[name] = up_rows(held, *w, k, junk=junk)
            self.host[name] = mx.decode(*w, k).reshape(n, rows, k)


def step(gpu, held, stack, x, dtype, sel, wts, resid, ld=None, rule=None, in_place=False):
    m, top_k = sel.shape
    hidden, ff = stack.hidden, stack.ff
    ld = ld or hidden
    xd = held.up(lines(x, dtype, ld, np.nan))
    rd = None if resid is None else held.up(lines(resid, dtype, ld + 1, np.nan))
    work = held.out(np.uint8, bm.mx4_moe_work(m, top_k, hidden, ff), 0xFF)
    y = rd if in_place else held.out(NUMPY[dtype], m * (ld + 1))
    gpu.enqueue_mx4_moe(stack.dev["gate"], stack.dev["up"], stack.dev["down"], stack.n, hidden, ff, xd, dtype, m, held.up(sel), held.up(wts.astype(np.float32)), top_k,
                        rd, y, work, ld_x=ld, ld_resid=ld + 1, ld_y=ld + 1, rule=rule)
    got = y.download().reshape(m, ld + 1)
    if not in_place:
        assert (got[:, hidden:].view(np.uint8) == 0xEE).all()
    return got[:, :hidden]


def assert_step(got, dtype, stack, x, sel, wts, resid):
    assert_near(got, dtype, *mx.moe(x, sel, wts.astype(np.float32), stack.host["gate"], stack.host["up"], stack.host["down"], stack.n, resid, KEPT[dtype]))


MOE = ((1, 1, 1, 1, 1), (1, 4, 2, 32, 32), (1, 4, 4, 33, 31), (2, 8, 3, 100, 70), (1, 16, 8, 512, 256), (3, 5, 5, 300, 513), (16, 8, 8, 256, 96), (5, 64, 8, 1000, 160),
       (17, 3, 2, 544, 64), (64, 16, 4, 160, 128), (64, 2, 2, 96, 300), (33, 40, 1, 64, 1100), (1, 3, 2, 2048, 768), (2, 1, 1, 4100, 40))


@DTYPES
@pytest.mark.parametrize("m,n,top_k,hidden,ff", MOE)
def test_the_experts_step(gpu, held, dtype, m, n, top_k, hidden, ff):
    rng = np.random.default_rng(3000 + m + hidden + ff)
    stack = Stack(held, rng, n, hidden, ff)
    x, resid = (rounded(normal_f32(rng, (m, hidden)), dtype) for _ in range(2))
    sel, wts = picks(rng, m, n, top_k, 0.1), rng.random((m, top_k)).astype(np.float32)
    got = step(gpu, held, stack, x, dtype, sel, wts, resid, ld=hidden + 3)
    assert_step(got, dtype, stack, x, sel, wts, resid)
    clean(gpu)


@pytest.mark.parametrize("m,top_k", ((3, 4), (20, 8)))
def test_no_residual_and_onto_the_residual(gpu, held, m, top_k):
    rng = np.random.default_rng(31)
    stack = Stack(held, rng, 6, 128, 96)
    x, resid = normal_f32(rng, (m, 128)), normal_f32(rng, (m, 128))
    sel, wts = picks(rng, m, 6, top_k), rng.random((m, top_k)).astype(np.float32)
    assert_step(step(gpu, held, stack, x, bm.F32, sel, wts, None), bm.F32, stack, x, sel, wts, None)
    assert_step(step(gpu, held, stack, x, bm.F32, sel, wts, resid, in_place=True), bm.F32, stack, x, sel, wts, resid)
    clean(gpu)


@DTYPES
def test_slots_served_elsewhere_past_the_stack_and_twice_the_same(gpu, held, dtype):
    rng = np.random.default_rng(32)
    m, n, top_k, hidden, ff = 9, 5, 4, 200, 130
    stack = Stack(held, rng, n, hidden, ff)
    x, resid = (rounded(normal_f32(rng, (m, hidden)), dtype) for _ in range(2))
    sel, wts = picks(rng, m, n, top_k), rng.random((m, top_k)).astype(np.float32)
    sel[0] = bm.HOST_SLOT                       # nothing of this token is here
    sel[1] = [3, 3, 3, 3]                       # one expert at every slot
    sel[2] = [bm.HOST_SLOT, 4, bm.HOST_SLOT, 4]
    sel[5:] = 1                                 # most tokens the same expert
    wts[1, 2] = 0.0
    wts[0] = np.nan                             # weights of slots that add nothing are not looked at
    wts[2, 0] = np.inf
    clean_wts = np.where(sel == bm.HOST_SLOT, 0, wts)
    got = step(gpu, held, stack, x, dtype, sel, wts, resid)
    assert_step(got, dtype, stack, x, sel, clean_wts, resid)
    assert np.array_equal(values(got[0], dtype), resid[0])
    clean(gpu)
    sel[3, 1], sel[4, 0], wts[3, 1] = n, 0xFFFFFFFE, np.nan
    got = step(gpu, held, stack, x, dtype, sel, wts, resid)
    assert_step(got, dtype, stack, x, sel, np.where(sel >= n, 0, wts), resid)
    assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    gpu.fault_clear()


@pytest.mark.parametrize("rule", range(1, len(RULES)))
def test_the_step_under_other_rules(gpu, held, rule):
    rng = np.random.default_rng(33)
    m, n, top_k, hidden, ff = 3, 4, 2, 128, 64
    stack = Stack(held, rng, n, hidden, ff)
    x, sel, wts = normal_f32(rng, (m, hidden)), picks(rng, m, n, top_k), rng.random((m, top_k)).astype(np.float32)
    got = values(step(gpu, held, stack, x, bm.F32, sel, wts, None, rule=RULES[rule][0]), bm.F32)
    want, size = np.zeros((m, hidden)), np.zeros((m, hidden))
    for t in range(m):
        for s in range(top_k):
            e = sel[t, s]
            h = RULES[rule][1](stack.host["gate"][e] @ x[t], stack.host["up"][e] @ x[t])
            want[t] += wts[t, s] * (stack.host["down"][e] @ h)
            size[t] += wts[t, s] * (np.abs(stack.host["down"][e]) @ (np.abs(h) + 1))
    assert (np.abs(got - want) <= 2.0 ** -16 * size).all()  # a rule's slopes are below 27: 76 steps of a sum times 27 of 2^-23
    clean(gpu)


def test_a_gate_that_is_not_finite_under_a_clamped_rule(gpu, held):
    rng = np.random.default_rng(34)
    stack = Stack(held, rng, 2, 64, 64)
    x = normal_f32(rng, (2, 64))
    x[1, 5] = np.inf
    sel, wts = np.array([[0], [1]], np.uint32), np.ones((2, 1), np.float32)
    gpu.fault_clear()
    got = values(step(gpu, held, stack, x, bm.F32, sel, wts, None, rule=(bm.ACT_SWIGLU_CLAMP, 1.0)), bm.F32)
    assert np.isfinite(got[0]).all() and np.isnan(got[1]).any()
    assert gpu.fault()[0] & 0xFF == bm.SITE_F32_PRODUCT
    gpu.fault_clear()


# ------------------------------------------------------------------------------------------- a layer of them

def test_a_layer_in_blocks_from_router_to_residual(gpu, held):
    """Router, sort, gate and up over shared columns, SwiGLU, down, and back onto the residual; and the whole step from the same ids; eager,
    then captured and replayed over other rows. Every stage is checked from the stage before it as the device left it."""
    rng = np.random.default_rng(14)
    m, hidden, ff, n, top_k = 37, 256, 192, 16, 4
    dtype = bm.BF16
    stack = Stack(held, rng, n, hidden, ff)
    rd = held.up(normal_f32(rng, (n, hidden)) * np.float32(0.1))
    xf, xb = held.out(np.float32, m * hidden), held.out(np.uint16, m * hidden)
    logits, ids, wts = held.out(np.float32, m * n), held.out(np.uint32, m * top_k), held.out(np.float32, m * top_k)
    slots = m * top_k
    order, start, place = held.out(np.uint32, slots), held.out(np.uint32, n + 1), held.out(np.uint32, slots)
    codes, scales = held.out(np.uint8, m * mx.row_bytes(hidden)), held.out(np.uint8, m * mx.row_scales(hidden))
    g, u = held.out(np.uint16, slots * ff), held.out(np.uint16, slots * ff)
    hc, hs = held.out(np.uint8, slots * mx.row_bytes(ff)), held.out(np.uint8, slots * mx.row_scales(ff))
    d, y, z = held.out(np.uint16, slots * hidden), held.out(np.uint16, m * hidden), held.out(np.uint16, m * hidden)
    work = held.out(np.uint8, bm.mx4_moe_work(m, top_k, hidden, ff))

    def enqueue():
        gpu.enqueue_router_logits(rd, xf, None, 1e-6, m, n, hidden, None, logits)
        gpu.enqueue_route_softmax(logits, m, n, top_k, True, None, ids, wts)
        gpu.enqueue_expert_sort(ids, m, top_k, n, None, dtype, 0, order, start, place, None)
        gpu.enqueue_mx4_quantize(xb, dtype, m, hidden, codes, scales)
        for name, out in (("gate", g), ("up", u)):
            gpu.enqueue_mx4_gemm_experts(*stack.dev[name], n, ff, hidden, codes, scales, order, start, slots, top_k, out, dtype)
        gpu.enqueue_mx4_swiglu_quantize(g, u, dtype, slots, ff, hc, hs, live=start.ptr + 4 * n)
        gpu.enqueue_mx4_gemm_experts(*stack.dev["down"], n, hidden, ff, hc, hs, order, start, slots, 0, d, dtype)
        gpu.enqueue_expert_combine(d, dtype, place, wts, xb, m, top_k, hidden, y)
        gpu.enqueue_mx4_moe(stack.dev["gate"], stack.dev["up"], stack.dev["down"], n, hidden, ff, xb, dtype, m, ids, wts, top_k, xb, z, work)

    graph = None
    try:
        for turn in range(4):
            x = rounded(normal_f32(rng, (m, hidden)), dtype)
            xf.upload(x.astype(np.float32))
            xb.upload(bits(x, dtype))
            y.fill_bytes(0xEE)
            z.fill_bytes(0xEE)
            if turn == 1:
                gpu.capture_begin()
                enqueue()
                graph = gpu.capture_end()
            if turn == 0:
                enqueue()
            else:
                gpu.graph_launch(graph)
            clean(gpu)
            picked, weights = ids.download().reshape(m, top_k), wts.download().reshape(m, top_k)
            want_order, want_start, want_place = tables(picked, n)
            assert np.array_equal(order.download(), want_order) and np.array_equal(start.download(), want_start)
            assert_rows(codes, scales, x)
            xv = mx.decode(*mx.encode(x), hidden)
            expert, col = np.repeat(np.arange(n), np.diff(want_start.astype(np.int64))), want_order // top_k
            for name, out in (("gate", g), ("up", u)):
                got = out.download().reshape(slots, ff)
                for e in range(n):
                    at = np.flatnonzero(expert == e)
                    if at.size:
                        assert_near(got[at], dtype, *mx.product_bound(xv[col[at]], stack.host[name][e]))
            hv = mx.decode(*mx.unpack(hc.download().reshape(slots, -1), hs.download().reshape(slots, -1), ff), ff)
            gv, uv = values(g.download(), dtype).reshape(slots, ff), values(u.download(), dtype).reshape(slots, ff)
            h = mx.rule_value(gv, uv)
            most = np.abs(h).reshape(slots, -1, 32).max(axis=2).repeat(32, axis=1)
            assert (np.abs(hv - h) <= most * 0.25).all()  # half of the widest step, 2 of 4; a block's largest value may be cut from 8 to 6
            got = d.download().reshape(slots, hidden)
            for e in range(n):
                at = np.flatnonzero(expert == e)
                if at.size:
                    assert_near(got[at], dtype, *mx.product_bound(hv[at], stack.host["down"][e]))
            terms = values(got, dtype).reshape(slots, hidden)[want_place].reshape(m, top_k, hidden) * weights.astype(np.float64)[:, :, None]
            bound = (top_k + 1) * 2.0 ** -24 * (np.abs(terms).sum(axis=1) + np.abs(x))
            assert_near(y.download().reshape(m, hidden), dtype, x + terms.sum(axis=1), bound)
            assert_step(z.download().reshape(m, hidden), dtype, stack, x, picked, weights, x)
    finally:
        if graph is not None:
            gpu.graph_destroy(graph)


def test_on_a_stream_of_torchs(held):
    """A context on torch's own stream: the launches stand in line with torch's work there."""
    rng = np.random.default_rng(15)
    stream = torch.cuda.Stream()
    own = bm.Gpu(0, stream=stream.cuda_stream)
    try:
        w = some_rows_zeroed(rng, 128, 256)
        words, padded = mx.pack(*w, 256)
        with torch.cuda.stream(stream):
            x = torch.randn(40, 256, device="cuda")
            wt, wst = torch.from_numpy(words).cuda(), torch.from_numpy(padded).cuda()
            codes, scales = torch.zeros(40, 128, dtype=torch.uint8, device="cuda"), torch.zeros(40, 16, dtype=torch.uint8, device="cuda")
            y = torch.zeros(40, 128, dtype=torch.float16, device="cuda")
            for _ in range(3):
                x = x * 2.0 + 1.0
                own.enqueue_mx4_gemm_x(wt.data_ptr(), wst.data_ptr(), 128, 256, x.data_ptr(), bm.F32, 40, codes.data_ptr(), scales.data_ptr(),
                                       y.data_ptr(), bm.F16)
                z = y * 1.0
        stream.synchronize()
        xv = mx.decode(*mx.encode(x.cpu().numpy()), 256)
        assert_near(z.cpu().view(torch.int16).numpy().view(np.uint16), bm.F16, *mx.product_bound(xv, mx.decode(*w, 256)))
    finally:
        own.close()
