"""GPU tests of the products in 8-bit integers (bm_i8_quantize, bm_i8_swiglu_quantize, bm_i8_gemm, bm_i8_gemm_x, bm_i8_gemm_experts)
against plain numpy: codes and scales exactly, by the rule's quotients in 64 bits; products bit for bit, from int64 sums and the
rule's three f32 roundings, and within those roundings of the value in 64 bits."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
from common import normal_f32
from rows_common import HALF_STEP, NAMES, NUMPY, TORCH, bits, codes_of, lines, padded, product, rounded, tables, values

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
        return self.keep(self.gpu.upload(host))

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


def quantize(gpu, held, x, dtype, k, ld=None, live=None):
    """Codes (padded rows) and scales of the host rows x; what lies between rows of a longer line is a NaN."""
    m = x.shape[0]
    xd = held.up(lines(x, dtype, ld or k, np.nan))
    kp = bm.i8_row_bytes(k)
    codes, scales = held.out(np.int8, m * kp, 0x55), held.out(np.float32, m)
    gpu.enqueue_i8_quantize(xd, dtype, m, k, codes, scales, ld_x=ld, live=live)
    return codes, scales


# ------------------------------------------------------------------------------------------------ quantizer

@DTYPES
@pytest.mark.parametrize("m,k,ld", ((1, 1, 1), (5, 2, 3), (7, 15, 15), (6, 16, 16), (9, 17, 19), (5, 500, 500), (5, 512, 515), (3, 513, 513),
                                    (4, 1024, 1024), (3, 1030, 1031), (5, 2048, 2048), (3, 2049, 2052), (3, 4096, 4096), (2, 5000, 5001),
                                    (2, 8192, 8192), (2, 8200, 8200), (1, 30001, 30001), (257, 64, 64)))
def test_codes_are_the_rules(gpu, held, dtype, m, k, ld):
    rng = np.random.default_rng(100 + m + k)
    x = rounded(normal_f32(rng, (m, k)) * np.exp(normal_f32(rng, (m, 1))), dtype)
    codes, scales = quantize(gpu, held, x, dtype, k, ld)
    q, s = codes_of(x)
    assert np.array_equal(scales.download(), s)
    assert np.array_equal(codes.download().reshape(m, -1), padded(q, k))
    clean(gpu)


def test_halves_go_to_even_and_their_neighbours_to_the_nearer(gpu, held):
    """Rows whose scale is a power of two hold exact halves; their f32 neighbours on either side are next to them."""
    half = np.arange(-126.5, 127.0, 1.0, np.float32)
    rows = []
    for e in (0, -3, 40, -60, -70, -120, 100):  # scales 2^e: both sides of where small scales are lifted
        v = np.concatenate([half, np.nextafter(half, np.float32(1e9)), np.nextafter(half, np.float32(-1e9)), [127.0]]).astype(np.float32)
        rows.append(v * np.float32(2.0) ** e)
    # and of a scale that is none: quotients as near a half as f32 values come
    for amax in (1.0, 0.7, 3e-5, 12345.678):
        s = np.float32(amax) / np.float32(127.0)
        v = (half.astype(np.float64) * np.float64(s)).astype(np.float32)
        rows.append(np.concatenate([v, np.nextafter(v, np.float32(1e9)), np.nextafter(v, np.float32(-1e9)), [np.float32(amax)]]).astype(np.float32))
    x = np.stack(rows)
    codes, scales = quantize(gpu, held, x, bm.F32, x.shape[1])
    q, s = codes_of(x)
    assert np.array_equal(scales.download(), s)
    assert np.array_equal(codes.download().reshape(x.shape[0], -1), padded(q, x.shape[1]))
    clean(gpu)


def test_small_large_and_empty_rows(gpu, held):
    tiny = np.float32(2.0 ** -149)
    rows = np.zeros((9, 40), np.float32)
    rows[1, 3] = -0.0
    rows[2, :5] = [tiny * 60, -tiny, 0, tiny, tiny * 59]           # the scale rounds to zero
    rows[3, :5] = [tiny * 64, -tiny, 0, tiny, tiny * 63]           # to the smallest
    rows[4, :5] = [tiny * 190, -tiny * 189, tiny * 100, tiny, 0]   # a quotient past 127
    rows[5, :4] = [3.4028235e38, -3.4e38, 1.0, 1e38]
    rows[6, :3] = [2.0 ** -126, 2.0 ** -130, -2.0 ** -127]
    rows[7, :] = -5.0
    rows[8, 39] = 1e-30
    codes, scales = quantize(gpu, held, rows, bm.F32, 40)
    q, s = codes_of(rows)
    assert np.array_equal(scales.download(), s)
    assert np.array_equal(codes.download().reshape(9, -1), padded(q, 40))
    clean(gpu)


@pytest.mark.parametrize("k", (40, 700, 2000, 9000))
@pytest.mark.parametrize("value", (np.nan, np.inf, -np.inf))
def test_a_row_that_is_not_finite(gpu, held, k, value):
    rng = np.random.default_rng(7)
    x = normal_f32(rng, (4, k))
    x[1, k - 1] = value
    gpu.fault_clear()
    codes, scales = quantize(gpu, held, x, bm.F32, k)
    got, s = codes.download().reshape(4, -1), scales.download()
    assert np.isnan(s[1]) and not got[1].any()
    q, want = codes_of(x)
    assert np.array_equal(np.delete(s, 1), np.delete(want, 1)) and np.array_equal(got, padded(q, k))
    assert gpu.fault()[0] & 0xFF == bm.SITE_QUANT_COLUMN
    gpu.fault_clear()


@pytest.mark.parametrize("k", (48, 2048, 9000))
def test_rows_behind_the_live_ones_keep_what_they_held(gpu, held, k):
    rng = np.random.default_rng(8)
    x = normal_f32(rng, (6, k))
    for live in (0, 1, 4, 6, 1000):
        codes, scales = quantize(gpu, held, x, bm.F32, k, live=held.up(np.array([live], np.uint32)))
        n = min(live, 6)
        q, s = codes_of(x)
        assert np.array_equal(codes.download().reshape(6, -1)[:n], padded(q, k)[:n]) and np.array_equal(scales.download()[:n], s[:n])
        assert (codes.download().reshape(6, -1)[n:] == 0x55).all() and (scales.download()[n:].view(np.uint32) == 0xEEEEEEEE).all()
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("rule", ((bm.ACT_SILU_MUL, 0.0), (bm.ACT_SWIGLU_CLAMP, 1.5), (bm.ACT_SWIGLU_OAI, 2.0), (bm.ACT_SITU, 3.0),
                                  (bm.ACT_SWIGLU_GCLAMP, 1.0)))
def test_the_gate_rules_values_quantized(gpu, held, dtype, rule):
    """h's relative error against 64 bits: the exponential and the divide are within a few units in the last place (64 x 2^-24 taken),
    the tanh of SiTU within 1e-5 (the entry's contract), so a scale is within that and a code within one step, and only where the
    quotient lies within that of a half."""
    import math
    rng = np.random.default_rng(9)
    m, k, ld = 5, 300, 303
    g, u = rounded(normal_f32(rng, (m, k)) * 2, dtype), rounded(normal_f32(rng, (m, k)), dtype)
    gd, ud = held.up(lines(g, dtype, ld, np.nan)), held.up(lines(u, dtype, ld, np.nan))
    codes, scales = held.out(np.int8, m * bm.i8_row_bytes(k)), held.out(np.float32, m)
    gpu.enqueue_i8_swiglu_quantize(gd, ud, dtype, m, k, codes, scales, ld=ld, rule=rule)
    sig = 1 / (1 + np.exp(-g))
    lim = rule[1]
    h = {bm.ACT_SILU_MUL: lambda: g * sig * u, bm.ACT_SWIGLU_CLAMP: lambda: np.minimum(g * sig, lim) * np.clip(u, -lim, lim),
         bm.ACT_SWIGLU_OAI: lambda: np.minimum(g, lim) / (1 + np.exp(-1.702 * np.minimum(g, lim))) * (np.clip(u, -lim, lim) + 1),
         bm.ACT_SITU: lambda: lim * np.tanh(g / lim) * sig * 25 * np.tanh(u / 25),
         bm.ACT_SWIGLU_GCLAMP: lambda: np.minimum(g, lim) / (1 + np.exp(-np.minimum(g, lim))) * np.clip(u, -lim, lim)}[rule[0]]()
    tol = 1e-5 if rule[0] == bm.ACT_SITU else 64 * 2.0 ** -24
    amax = np.abs(h).max(axis=1)
    assert np.allclose(scales.download(), amax / 127, rtol=tol + 2.0 ** -23, atol=0)
    got = codes.download().reshape(m, -1)
    quotient = h / (amax / 127)[:, None]
    # amax and h both off by tol at most: the quotient by twice that of at most 127
    assert (np.abs(got[:, :k] - quotient) <= 0.5 + 127 * (2 * tol + 2.0 ** -22)).all()
    assert not got[:, k:].any()
    clean(gpu)
    # the context's rule where the launch has none of its own
    gpu.set_gate_rule(*rule)
    again, s2 = held.out(np.int8, m * bm.i8_row_bytes(k)), held.out(np.float32, m)
    gpu.enqueue_i8_swiglu_quantize(gd, ud, dtype, m, k, again, s2, ld=ld)
    gpu.set_gate_rule(bm.ACT_SILU_MUL)
    assert np.array_equal(again.download(), codes.download()) and np.array_equal(s2.download(), scales.download())


def test_a_gate_that_is_not_finite(gpu, held):
    for rule, sites in (((bm.ACT_SILU_MUL, 0.0), 1 << bm.SITE_QUANT_COLUMN),
                        ((bm.ACT_SWIGLU_CLAMP, 1.0), (1 << bm.SITE_QUANT_COLUMN) | (1 << bm.SITE_F32_PRODUCT))):
        g, u = np.ones((3, 64), np.float32), np.ones((3, 64), np.float32)
        g[1, 5] = np.nan
        gpu.fault_clear()
        codes, scales = held.out(np.int8, 3 * 64), held.out(np.float32, 3)
        gpu.enqueue_i8_swiglu_quantize(held.up(g), held.up(u), bm.F32, 3, 64, codes, scales, rule=rule)
        s = scales.download()
        assert np.isnan(s[1]) and np.isfinite(s[[0, 2]]).all() and not codes.download().reshape(3, 64)[1].any()
        assert gpu.fault()[1] == sites
    gpu.fault_clear()


# ------------------------------------------------------------------------------------------------- products

def some_matrix(rng, rows, k):
    w = rng.integers(-128, 128, (rows, k), dtype=np.int16).astype(np.int8)
    return w, (rng.random(rows).astype(np.float32) + np.float32(0.5)) * np.float32(1e-3)


def junk_padded(w, k, rng):
    """Rows of a matrix with anything behind the k-th byte."""
    out = rng.integers(-128, 128, (w.shape[0], -(-k // 16) * 16), dtype=np.int16).astype(np.int8)
    out[:, :k] = w
    return out


def assert_product(words, want, dtype, exact, what=""):
    """Bits of the rule's f32 value rounded once; and near the value in 64 bits: three f32 roundings and the type's."""
    assert np.array_equal(words, bits(want, dtype)), f"{what}: {np.count_nonzero(words != bits(want, dtype))} of {words.size} values differ"
    got = values(words, dtype).reshape(exact.shape)
    # an f16 below its normal range is off by half its smallest step
    assert (np.abs(got - exact) <= (HALF_STEP[dtype] + 3.1 * 2.0 ** -24) * np.abs(exact) + (2.0 ** -25 if dtype == bm.F16 else 0)).all(), what


SIZES = ((1, 1, 1), (1, 768, 2048), (2, 5, 16), (3, 17, 63), (4, 16, 64), (5, 100, 65), (8, 256, 128), (15, 33, 130), (16, 64, 192), (17, 255, 256),
         (31, 257, 100), (32, 128, 1024), (33, 129, 1040), (48, 70, 2056), (64, 512, 384), (65, 300, 129), (100, 640, 512), (127, 128, 640),
         (128, 256, 768), (129, 257, 272), (200, 1000, 333), (256, 256, 256), (257, 513, 1000), (300, 2000, 1996), (513, 384, 896), (1030, 260, 144))


@DTYPES
@pytest.mark.parametrize("m,rows,k", SIZES)
def test_product_of_rows_of_any_size(gpu, held, dtype, m, rows, k):
    rng = np.random.default_rng(1000 + 7 * m + rows + k)
    w, ws = some_matrix(rng, rows, k)
    x = rounded(normal_f32(rng, (m, k)), dtype)
    q, s = codes_of(x)
    want = product(q, s, w, ws)
    exact = (q.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64) * s.astype(np.float64)[:, None] * ws.astype(np.float64)
    wd, wsd = held.up(junk_padded(w, k, rng)), held.up(ws)
    codes, scales = quantize(gpu, held, x, dtype, k)
    ld = rows + 3
    y = held.out(NUMPY[dtype], m * ld)
    gpu.enqueue_i8_gemm(wd, wsd, rows, k, codes, scales, m, y, dtype, ld_y=ld)
    got = y.download().reshape(m, ld)
    assert_product(got[:, :rows], want, dtype, exact, "bm_i8_gemm")
    assert (got[:, rows:].view(np.uint8) == 0xEE).all(), "written between the rows"
    # and from the rows in one call, into rows back to back
    c2, s2, y2 = held.out(np.int8, m * bm.i8_row_bytes(k), 0x33), held.out(np.float32, m), held.out(NUMPY[dtype], m * rows)
    gpu.enqueue_i8_gemm_x(wd, wsd, rows, k, held.up(lines(x, dtype, k + 5, np.nan)), dtype, m, c2, s2, y2, dtype, ld_x=k + 5)
    assert np.array_equal(y2.download().reshape(m, rows), got[:, :rows])
    assert np.array_equal(c2.download(), codes.download()) and np.array_equal(s2.download(), scales.download())
    clean(gpu)


@pytest.mark.parametrize("m", (1, 20, 130))
def test_the_longest_rows_do_not_overflow(gpu, held, m):
    k, rows = 131072, 3
    w = np.full((rows, k), -128, np.int8)
    w[1] = 127
    w[2, ::2] = 127
    q = np.full((m, k), 127, np.int8)
    s, ws = np.ones(m, np.float32), np.ones(rows, np.float32)
    y = held.out(np.float32, m * rows)
    gpu.enqueue_i8_gemm(held.up(w), held.up(ws), rows, k, held.up(q), held.up(s), m, y, bm.F32)
    assert np.array_equal(y.download().reshape(m, rows), product(q, s, w, ws))


@pytest.mark.parametrize("m", (1, 3, 40, 300))
def test_a_row_that_is_not_finite_reaches_its_own_outputs_only(gpu, held, m):
    rng = np.random.default_rng(11)
    k, rows = 320, 200
    x = normal_f32(rng, (m, k))
    x[m // 2, 7] = np.inf
    w, ws = some_matrix(rng, rows, k)
    gpu.fault_clear()
    y = held.out(np.float32, m * rows)
    codes, scales = held.out(np.int8, m * k), held.out(np.float32, m)
    gpu.enqueue_i8_gemm_x(held.up(w), held.up(ws), rows, k, held.up(x), bm.F32, m, codes, scales, y, bm.F32)
    got = y.download().reshape(m, rows)
    assert np.isnan(got[m // 2]).all() and np.isfinite(np.delete(got, m // 2, 0)).all()
    assert gpu.fault()[0] & 0xFF == bm.SITE_QUANT_COLUMN
    gpu.fault_clear()


def test_other_types_of_output_than_of_input(gpu, held):
    rng = np.random.default_rng(12)
    w, ws = some_matrix(rng, 100, 256)
    for m in (1, 3, 50, 260):
        x = rounded(normal_f32(rng, (m, 256)), bm.BF16)
        q, s = codes_of(x)
        want = product(q, s, w, ws)
        for t in (bm.F32, bm.F16):
            y = held.out(NUMPY[t], m * 100)
            gpu.enqueue_i8_gemm_x(held.up(w), held.up(ws), 100, 256, held.up(bits(x, bm.BF16)), bm.BF16, m, held.out(np.int8, m * 256),
                                  held.out(np.float32, m), y, t)
            assert np.array_equal(y.download().reshape(m, 100), bits(want, t))
    clean(gpu)


# --------------------------------------------------------------------------------------- products of experts

def picks(rng, m, n, top_k, away=0.2):
    ids = np.stack([rng.permutation(n)[:top_k] for _ in range(m)]).astype(np.uint32)
    ids[rng.random(ids.shape) < away] = bm.HOST_SLOT
    return ids


@DTYPES
@pytest.mark.parametrize("m,n,top_k,rows,k", ((1, 4, 2, 16, 16), (1, 1, 1, 5, 40), (3, 8, 8, 33, 130), (16, 64, 8, 768, 256), (5, 300, 4, 20, 64),
                                              (40, 6, 3, 257, 320), (200, 5, 2, 130, 192), (150, 3, 3, 300, 1000), (700, 4, 2, 256, 512)))
def test_experts_product_over_shared_and_own_columns(gpu, held, dtype, m, n, top_k, rows, k):
    rng = np.random.default_rng(2000 + m + rows)
    ids = picks(rng, m, n, top_k)
    if n > 4:
        ids[ids == 2] = bm.HOST_SLOT  # an expert that nobody picked
    order, start, _ = tables(ids, n)
    n_slots, listed = m * top_k, int(start[-1])
    w, ws = some_matrix(rng, n * rows, k)
    full = np.full(n_slots, 0x12345678, np.uint32)  # behind the listed entries: what no launch may follow
    full[:listed] = order
    wd, wsd, od, sd = held.up(junk_padded(w, k, rng)), held.up(ws), held.up(full), held.up(start)
    w3, ws2 = w.reshape(n, rows, k), ws.reshape(n, rows)
    expert = np.repeat(np.arange(n), np.diff(start.astype(np.int64)))
    for own in (False, True):
        x = rounded(normal_f32(rng, (n_slots if own else m, k)), dtype)
        q, s = codes_of(x)
        codes, scales = quantize(gpu, held, x, dtype, k)
        col = np.arange(listed) if own else order // top_k
        ld = rows + 1
        y = held.out(NUMPY[dtype], n_slots * ld)
        gpu.enqueue_i8_gemm_experts(wd, wsd, n, rows, k, codes, scales, None if own else od, sd, n_slots, 0 if own else top_k, y, dtype, ld_y=ld)
        got = y.download().reshape(n_slots, ld)
        for e in range(n):
            at = np.flatnonzero(expert == e)
            if at.size:
                qe, se = q[col[at]], s[col[at]]
                exact = (qe.astype(np.int64) @ w3[e].astype(np.int64).T).astype(np.float64) * se.astype(np.float64)[:, None] * ws2[e].astype(np.float64)
                assert_product(got[at, :rows], product(qe, se, w3[e], ws2[e]), dtype, exact, f"expert {e}")
        assert (got[listed:].view(np.uint8) == 0xEE).all() and (got[:, rows:].view(np.uint8) == 0xEE).all()
    clean(gpu)


@pytest.mark.parametrize("rows", (48, 300))
def test_tables_that_are_none_are_skipped(gpu, held, rows):
    """Runs that run backwards or past the slots, entries that name no slot: raised, nothing out of range read or written."""
    rng = np.random.default_rng(13)
    n, k, n_slots, top_k = 4, 64, 12, 2
    w, ws = some_matrix(rng, n * rows, k)
    x = normal_f32(rng, (6, k))
    codes, scales = quantize(gpu, held, x, bm.F32, k)
    q, s = codes_of(x)
    order = np.arange(12, dtype=np.uint32)
    wd, wsd = held.up(w), held.up(ws)
    want = [product(q, s, w[e * rows:(e + 1) * rows], ws[e * rows:(e + 1) * rows]) for e in range(n)]
    for start, ok in (((0, 3, 2, 5, 12), {0: (0, 3), 2: (2, 5), 3: (5, 12)}), ((0, 3, 6, 9, 13), {0: (0, 3), 1: (3, 6), 2: (6, 9)}),
                      ((0, 3, 0xFFFFFFF0, 9, 12), {0: (0, 3), 3: (9, 12)})):
        gpu.fault_clear()
        y = held.out(np.float32, n_slots * rows)
        gpu.enqueue_i8_gemm_experts(wd, wsd, n, rows, k, codes, scales, held.up(order), held.up(np.array(start, np.uint32)), n_slots, top_k, y, bm.F32)
        got = y.download().reshape(n_slots, rows)
        if start[1] <= start[2]:  # runs that do not overlap
            done = np.zeros(n_slots, bool)
            for e, (a, b) in ok.items():
                assert np.array_equal(got[a:b], want[e][order[a:b] // top_k])
                done[a:b] = True
            assert (got[~done].view(np.uint32) == 0xEEEEEEEE).all()
        assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    bad = order.copy()
    bad[[1, 7]] = [12, 0xFFFFFFFF]
    gpu.fault_clear()
    y = held.out(np.float32, n_slots * rows)
    gpu.enqueue_i8_gemm_experts(wd, wsd, n, rows, k, codes, scales, held.up(bad), held.up(np.array((0, 3, 6, 9, 12), np.uint32)), n_slots, top_k, y, bm.F32)
    got = y.download().reshape(n_slots, rows)
    assert np.isnan(got[[1, 7]]).all() and np.isfinite(np.delete(got, [1, 7], 0)).all()
    assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    gpu.fault_clear()


# ------------------------------------------------------------------------------------------- a layer of them

def test_a_layer_of_eight_bit_experts_from_router_to_residual(gpu, held):
    """Router, sort, gate and up over shared columns, SwiGLU, down, and back onto the residual; eager, then captured and replayed over other
    rows. Every stage is checked from the stage before it as the device left it."""
    rng = np.random.default_rng(14)
    m, hidden, ff, n, top_k = 37, 256, 192, 16, 4
    dtype = bm.BF16
    router = normal_f32(rng, (n, hidden)) * 0.1
    mats = {name: some_matrix(rng, n * r, c) for name, r, c in (("gate", ff, hidden), ("up", ff, hidden), ("down", hidden, ff))}
    dev = {name: (held.up(w), held.up(s)) for name, (w, s) in mats.items()}
    rd = held.up(router)
    xf, xb = held.out(np.float32, m * hidden), held.out(np.uint16, m * hidden)
    logits, ids, wts = held.out(np.float32, m * n), held.out(np.uint32, m * top_k), held.out(np.float32, m * top_k)
    slots = m * top_k
    order, start, place = held.out(np.uint32, slots), held.out(np.uint32, n + 1), held.out(np.uint32, slots)
    codes, scales = held.out(np.int8, m * hidden), held.out(np.float32, m)
    g, u = held.out(np.uint16, slots * ff), held.out(np.uint16, slots * ff)
    hc, hs = held.out(np.int8, slots * ff), held.out(np.float32, slots)
    d, y = held.out(np.uint16, slots * hidden), held.out(np.uint16, m * hidden)

    def enqueue():
        gpu.enqueue_router_logits(rd, xf, None, 1e-6, m, n, hidden, None, logits)
        gpu.enqueue_route_softmax(logits, m, n, top_k, True, None, ids, wts)
        gpu.enqueue_expert_sort(ids, m, top_k, n, None, dtype, 0, order, start, place, None)
        gpu.enqueue_i8_quantize(xb, dtype, m, hidden, codes, scales)
        for name, out in (("gate", g), ("up", u)):
            gpu.enqueue_i8_gemm_experts(*dev[name], n, ff, hidden, codes, scales, order, start, slots, top_k, out, dtype)
        gpu.enqueue_i8_swiglu_quantize(g, u, dtype, slots, ff, hc, hs, live=start.ptr + 4 * n)
        gpu.enqueue_i8_gemm_experts(*dev["down"], n, hidden, ff, hc, hs, order, start, slots, 0, d, dtype)
        gpu.enqueue_expert_combine(d, dtype, place, wts, xb, m, top_k, hidden, y)

    graph = None
    try:
        for turn in range(4):
            x = rounded(normal_f32(rng, (m, hidden)), dtype)
            xf.upload(x.astype(np.float32))
            xb.upload(bits(x, dtype))
            y.fill_bytes(0xEE)
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
            assert np.array_equal(place.download(), want_place)
            q, s = codes_of(x)
            expert, col = np.repeat(np.arange(n), np.diff(want_start.astype(np.int64))), want_order // top_k
            for name, out in (("gate", g), ("up", u)):
                w, ws = mats[name][0].reshape(n, ff, hidden), mats[name][1].reshape(n, ff)
                want = np.concatenate([product(q[col[expert == e]], s[col[expert == e]], w[e], ws[e]) for e in range(n)])
                assert np.array_equal(out.download().reshape(slots, ff), bits(want, dtype))
            gv, uv = values(g.download(), dtype).reshape(slots, ff), values(u.download(), dtype).reshape(slots, ff)
            h = gv / (1 + np.exp(-gv)) * uv
            got_hc, got_hs = hc.download().reshape(slots, ff), hs.download()
            amax = np.abs(h).max(axis=1)
            assert np.allclose(got_hs, amax / 127, rtol=2.0 ** -17, atol=0)
            assert (np.abs(got_hc - h / (amax / 127)[:, None]) <= 0.5 + 127 * 2.0 ** -16).all()
            w, ws = mats["down"][0].reshape(n, hidden, ff), mats["down"][1].reshape(n, hidden)
            want = np.concatenate([product(got_hc[expert == e], got_hs[expert == e], w[e], ws[e]) for e in range(n)])
            assert np.array_equal(d.download().reshape(slots, hidden), bits(want, dtype))
            dv = values(d.download(), dtype).reshape(slots, hidden)[want_place].reshape(m, top_k, hidden)
            terms = dv * weights.astype(np.float64)[:, :, None]
            exact = x + terms.sum(axis=1)
            got = values(y.download(), dtype).reshape(m, hidden)
            # an f32 rounding a term and one for the residual, of partial sums no larger than the terms' magnitudes; the type's at the end
            bound = (top_k + 1) * 2.0 ** -24 * (np.abs(terms).sum(axis=1) + np.abs(x))
            assert (np.abs(got - exact) <= HALF_STEP[dtype] * (np.abs(exact) + bound) + bound).all()
    finally:
        if graph is not None:
            gpu.graph_destroy(graph)


def test_on_a_stream_of_torchs(held):
    """A context on torch's own stream: the launches stand in line with torch's work there."""
    rng = np.random.default_rng(15)
    stream = torch.cuda.Stream()
    own = bm.Gpu(0, stream=stream.cuda_stream)
    try:
        w, ws = some_matrix(rng, 128, 256)
        with torch.cuda.stream(stream):
            x = torch.randn(40, 256, device="cuda")
            wt, wst = torch.from_numpy(w).cuda(), torch.from_numpy(ws).cuda()
            codes, scales = torch.zeros(40, 256, dtype=torch.int8, device="cuda"), torch.zeros(40, device="cuda")
            y = torch.zeros(40, 128, dtype=torch.float16, device="cuda")
            for _ in range(3):
                x = x * 2.0 + 1.0
                own.enqueue_i8_gemm_x(wt.data_ptr(), wst.data_ptr(), 128, 256, x.data_ptr(), bm.F32, 40, codes.data_ptr(), scales.data_ptr(),
                                      y.data_ptr(), bm.F16)
                z = y * 1.0
        stream.synchronize()
        q, s = codes_of(x.cpu().numpy())
        assert torch.equal(z.cpu(), torch.from_numpy(product(q, s, w, ws)).to(TORCH[bm.F16]))
    finally:
        own.close()
