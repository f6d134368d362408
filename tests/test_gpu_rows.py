"""GPU tests of tokens' rows sorted by expert and back (bm_expert_sort, bm_expert_combine and their gradients) against plain numpy: tables
and moved rows exactly; sums against 64 bits within their f32 roundings and the type's; gradients against the formulas and against
differences of the launches forward."""
import numpy as np
import pytest

import bloomery_amd as bm
from common import normal_f32
from rows_common import HALF_STEP, NAMES, NUMPY, bits, lines, rounded, tables, values
from test_gpu_i8 import clean, gpu, held, picks  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)
U32 = np.uint32


def sort(gpu, held, ids, n, x=None, dtype=bm.F32, pad=(0, 0)):
    """order, start, place and the moved rows' words, in buffers that held 0xEE bytes."""
    m, top_k = ids.shape
    slots = m * top_k
    order, start, place = held.out(U32, slots), held.out(U32, n + 1), held.out(U32, slots)
    need = bm.expert_sort_work(slots, n)
    work = held.out(U32, need) if need else None
    if x is None:
        gpu.enqueue_expert_sort(held.up(ids), m, top_k, n, None, 77, -1, order, start, place, None, work)
        return order.download(), start.download(), place.download(), None
    width = x.shape[1]
    rows = held.out(NUMPY[dtype], slots * (width + pad[1]))
    gpu.enqueue_expert_sort(held.up(ids), m, top_k, n, held.up(lines(x, dtype, width + pad[0], 7.0)), dtype, width, order, start, place, rows, work,
                            ld_x=width + pad[0], ld_rows=width + pad[1])
    return order.download(), start.download(), place.download(), rows.download().reshape(slots, width + pad[1])


def check_sort(got, ids, n, x, dtype, width):
    order, start, place, rows = got
    want_order, want_start, want_place = tables(ids, n)
    listed = want_order.size
    assert np.array_equal(start, want_start) and np.array_equal(place, want_place)
    assert np.array_equal(order[:listed], want_order) and (order[listed:] == 0xEEEEEEEE).all()
    if rows is not None:
        assert np.array_equal(rows[:listed, :width], bits(x, dtype)[want_order // ids.shape[1]])
        assert (rows[listed:].view(np.uint8) == 0xEE).all() and (rows[:, width:].view(np.uint8) == 0xEE).all()


@DTYPES
@pytest.mark.parametrize("m,n,top_k,width,pad", ((1, 1, 1, 1, (0, 0)), (1, 8, 8, 64, (0, 0)), (3, 5, 2, 7, (1, 2)), (16, 128, 8, 2048, (0, 0)),
                                                 (17, 1024, 3, 33, (0, 1)), (9, 64, 64, 129, (3, 0)), (300, 4, 2, 100, (0, 0)), (256, 16, 8, 40, (0, 0)),
                                                 (257, 16, 8, 40, (1, 1)), (1000, 128, 8, 24, (0, 0)), (2500, 1, 1, 9, (0, 3)), (700, 1024, 4, 17, (0, 0)),
                                                 (50, 100, 64, 5, (0, 0)), (512, 16, 8, 8, (0, 0)), (513, 16, 8, 9, (0, 1)), (5000, 1, 1, 3, (0, 0)),
                                                 (1500, 1024, 4, 8, (0, 0)), (2100, 130, 8, 16, (0, 0)), (150, 600, 40, 4, (0, 0)), (20000, 7, 7, 2, (0, 0)),
                                                 (7, 5, 1, 4100, (0, 1)), (4095, 64, 1, 20, (0, 0)), (1001, 9, 2, 300, (2, 0)), (9, 9, 2, 5003, (0, 0)), (1365, 20, 3, 12, (0, 0)), (6, 7, 5, 2100, (0, 0))))
def test_sort_is_the_stable_one(gpu, held, dtype, m, n, top_k, width, pad):
    rng = np.random.default_rng(m + n + width)
    ids = picks(rng, m, n, top_k)
    x = rounded(normal_f32(rng, (m, width)), dtype)
    check_sort(sort(gpu, held, ids, n, x, dtype, pad), ids, n, x, dtype, width)
    check_sort(sort(gpu, held, ids, n), ids, n, None, dtype, width)
    clean(gpu)


@pytest.mark.parametrize("m", (1, 40, 2000))
def test_sort_of_crowds_of_none_and_of_the_same_expert_twice(gpu, held, m):
    rng = np.random.default_rng(m)
    n, top_k, width = 6, 3, 20
    x = rounded(normal_f32(rng, (m, width)), bm.BF16)
    for ids in (np.full((m, top_k), 5), np.full((m, top_k), 0xFFFFFFFF), np.tile([[2, 2, 0]], (m, 1)), np.tile([[0xFFFFFFFF, 3, 0xFFFFFFFF]], (m, 1))):
        ids = ids.astype(U32)
        check_sort(sort(gpu, held, ids, n, x, bm.BF16), ids, n, x, bm.BF16, width)
    clean(gpu)


@pytest.mark.parametrize("m,top_k", ((1, 1), (20, 4), (1900, 4)))
def test_an_id_past_the_experts_raises_and_joins_no_run(gpu, held, m, top_k):
    rng = np.random.default_rng(3)
    ids = picks(rng, m, 8, top_k)
    ids[m // 2, 0] = 8
    if m > 1:
        ids[0, 1] = 0x80000000
    x = rounded(normal_f32(rng, (m, 12)), bm.F32)
    gpu.fault_clear()
    check_sort(sort(gpu, held, ids, 8, x), ids, 8, x, bm.F32, 12)
    assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    gpu.fault_clear()


def test_sorted_tables_are_the_buckets(gpu, held):
    rng = np.random.default_rng(4)
    for m, n, top_k in ((30, 17, 4), (3000, 256, 8)):
        ids = picks(rng, m, n, top_k)
        order, start, _, _ = sort(gpu, held, ids, n)
        o2, s2 = held.out(U32, m * top_k), held.out(U32, n + 1)
        gpu.enqueue_buckets(held.up(ids), m * top_k, n, o2, s2)
        assert np.array_equal(start, s2.download()) and np.array_equal(order, o2.download())
    clean(gpu)


class Rows:
    """A batch's picks, sorted rows, weights and rows at the tokens, on both sides."""

    def __init__(self, held, dtype, m, n, top_k, width, seed, pad=0, away=0.2):
        rng = np.random.default_rng(seed)
        self.m, self.top_k, self.width, self.dtype, self.ld = m, top_k, width, dtype, width + pad
        self.slots = m * top_k
        ids = picks(rng, m, n, top_k, away)
        if m > 2:
            ids[1] = bm.HOST_SLOT  # a token that is served elsewhere altogether
        self.place = tables(ids, n)[2]
        self.there = (self.place != 0xFFFFFFFF).reshape(m, top_k)
        self.listed = int(self.there.sum())
        self.rows = rounded(normal_f32(rng, (self.slots, width)), dtype)
        self.w = normal_f32(rng, (m, top_k))
        self.w[~self.there] = np.nan  # a weight that nobody may use
        self.tok = rounded(normal_f32(rng, (m, width)), dtype)
        rows = self.rows.copy()
        rows[self.listed:] = np.nan  # rows that nobody may use
        self.rows_d, self.place_d, self.w_d = held.up(lines(rows, dtype, self.ld, np.nan)), held.up(self.place), held.up(self.w)
        self.tok_d = held.up(lines(self.tok, dtype, self.ld, np.nan))
        at = np.where(self.there, self.place.reshape(m, top_k), 0).astype(np.int64)
        self.at = at
        self.mine = np.where(self.there[:, :, None], self.rows[at], 0.0)   # tokens x slots x width, f64
        self.w0 = np.where(self.there, self.w, 0.0).astype(np.float64)


BATCHES = ((1, 4, 1, 1, 0), (1, 8, 8, 2048, 0), (2, 16, 3, 7, 2), (5, 9, 9, 100, 0), (16, 128, 8, 2048, 0), (33, 64, 17, 513, 1), (3, 100, 64, 72, 0),
           (200, 8, 2, 24, 0), (40, 32, 8, 4100, 4), (77, 16, 4, 64, 0), (303, 9, 1, 425, 0), (50, 9, 1, 2100, 1), (50, 9, 2, 1024, 0),
           (50, 9, 2, 1030, 0), (21, 9, 4, 130, 3), (60, 12, 3, 2600, 0), (30, 12, 6, 500, 0))


def near(got, exact, terms, n_roundings, dtype):
    """n f32 roundings of partial sums no larger than the terms' magnitudes, then the type's rounding (f16: of subnormals too)."""
    bound = n_roundings * 2.0 ** -24 * terms
    assert (np.abs(got - exact) <= HALF_STEP[dtype] * (np.abs(exact) + bound) + bound + (2.0 ** -25 if dtype == bm.F16 else 0)).all()


@DTYPES
@pytest.mark.parametrize("m,n,top_k,width,pad", BATCHES)
def test_combine_and_the_sorts_gradient(gpu, held, dtype, m, n, top_k, width, pad):
    r = Rows(held, dtype, m, n, top_k, width, 50 + m + width, pad)
    for resid in (True, False):
        y = held.out(NUMPY[dtype], m * r.ld)
        gpu.enqueue_expert_combine(r.rows_d, dtype, r.place_d, r.w_d, r.tok_d if resid else None, m, top_k, width, y, ld_rows=r.ld, ld_resid=r.ld, ld_y=r.ld)
        words = y.download().reshape(m, r.ld)
        terms = r.mine * r.w0[:, :, None]
        base = r.tok if resid else 0.0 * r.tok
        near(values(words, dtype)[:, :width], base + terms.sum(1), np.abs(terms).sum(1) + np.abs(base), top_k + 1, dtype)
        assert (words[:, width:].view(np.uint8) == 0xEE).all()
    dx = held.out(NUMPY[dtype], m * r.ld)
    gpu.enqueue_expert_sort_grad(r.rows_d, dtype, r.place_d, m, top_k, width, dx, ld_rows=r.ld, ld_dx=r.ld)
    words = dx.download().reshape(m, r.ld)
    near(values(words, dtype)[:, :width], r.mine.sum(1), np.abs(r.mine).sum(1), top_k, dtype)
    assert (words[:, width:].view(np.uint8) == 0xEE).all()
    if m > 2:
        assert not values(words, dtype)[1, :width].any(), "a token with no listed slot"
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("m,n,top_k,width,pad", BATCHES)
def test_combines_gradients_are_the_formulas(gpu, held, dtype, m, n, top_k, width, pad):
    r = Rows(held, dtype, m, n, top_k, width, 80 + m + width, pad)
    d_rows, d_w = held.out(NUMPY[dtype], r.slots * r.ld), held.out(np.float32, r.slots)
    gpu.enqueue_expert_combine_grad(r.tok_d, dtype, r.rows_d, r.place_d, r.w_d, m, top_k, width, d_rows, d_w, ld_dy=r.ld, ld_rows=r.ld, ld_d_rows=r.ld)
    words = d_rows.download().reshape(r.slots, r.ld)
    got = values(words, dtype)[:, :width][r.at]
    exact = r.w0[:, :, None] * r.tok[:, None, :]
    for t in range(m):
        for k in range(top_k):
            if r.there[t, k]:
                near(got[t, k], exact[t, k], np.abs(exact[t, k]), 1, dtype)
    assert (words[r.listed:].view(np.uint8) == 0xEE).all() and (words[:, width:].view(np.uint8) == 0xEE).all()
    terms = r.mine * r.tok[:, None, :]
    # a dot is summed in any order: at most a rounding an addend along its longest chain, and no chain is longer than the row
    near(d_w.download().reshape(m, top_k).astype(np.float64), terms.sum(2), np.abs(terms).sum(2), width + 2, bm.F32)
    assert (d_w.download().reshape(m, top_k)[~r.there].view(U32) == 0).all()
    clean(gpu)


def test_the_f32_sum_is_combine_tokens_bit_for_bit(gpu, held):
    """Every slot listed, in slot order: the same terms in the same order as the sum over unsorted rows."""
    r = Rows(held, bm.F32, 20, 32, 8, 516, 5, away=0.0)
    rng = np.random.default_rng(6)
    place = rng.permutation(r.slots).astype(U32)
    w = normal_f32(rng, (20, 8))
    rows = normal_f32(rng, (r.slots, 516))
    y, y2 = held.out(np.float32, 20 * 516), held.out(np.float32, 20 * 516)
    gpu.enqueue_expert_combine(held.up(rows), bm.F32, held.up(place), held.up(w), r.tok_d, 20, 8, 516, y)
    gpu.enqueue_combine_tokens(held.up(rows[place]), held.up(w), r.tok_d, 516, 8, 20, y2)
    assert np.array_equal(y.download().view(U32), y2.download().view(U32))


@pytest.mark.parametrize("m,n,top_k,width", ((1, 4, 2, 40), (12, 16, 8, 300), (1100, 8, 4, 20)))
def test_gradients_against_differences(gpu, held, m, n, top_k, width):
    """Both maps are linear in their rows and in the weights, so a difference over a whole step D is the derivative along D: what the
    forward launches move by, against <gradient, D>. Tolerance: the f32 roundings of every sum on either side, in 64-bit dots."""
    rng = np.random.default_rng(m)
    ids = picks(rng, m, n, top_k)
    slots = m * top_k
    work = held.out(U32, max(1, bm.expert_sort_work(slots, n)))
    order, start, place = held.out(U32, slots), held.out(U32, n + 1), held.out(U32, slots)
    sel, w = held.up(ids), normal_f32(rng, (m, top_k))

    def forward(x):
        rows = held.out(np.float32, slots * width, 0)
        gpu.enqueue_expert_sort(sel, m, top_k, n, held.up(x), bm.F32, width, order, start, place, rows, work)
        return rows.download().reshape(slots, width).astype(np.float64)

    def back(rows, weights, resid):
        y = held.out(np.float32, m * width)
        gpu.enqueue_expert_combine(held.up(rows), bm.F32, place, held.up(weights), held.up(resid), m, top_k, width, y)
        return y.download().reshape(m, width).astype(np.float64)

    x, dx_step = normal_f32(rng, (m, width)), normal_f32(rng, (m, width))
    listed = int((ids != bm.HOST_SLOT).sum())
    g = normal_f32(rng, (slots, width))
    g[listed:] = 0
    dx = held.out(np.float32, m * width)
    moved = forward((x + dx_step).astype(np.float32)) - forward(x)
    gpu.enqueue_expert_sort_grad(held.up(g), bm.F32, place, m, top_k, width, dx)
    moved_by = ((x + dx_step).astype(np.float32).astype(np.float64) - x)
    want, terms = (dx.download().reshape(m, width).astype(np.float64) * moved_by), np.abs(g.astype(np.float64) * moved)
    assert abs((g * moved).sum() - want.sum()) <= top_k * 2.0 ** -24 * terms.sum() + 1e-12 * terms.sum()

    rows, row_step = normal_f32(rng, (slots, width)), normal_f32(rng, (slots, width))
    w_step, resid, dy = normal_f32(rng, (m, top_k)), normal_f32(rng, (m, width)), normal_f32(rng, (m, width))
    d_rows, d_w = held.out(np.float32, slots * width, 0), held.out(np.float32, slots)
    gpu.enqueue_expert_combine_grad(held.up(dy), bm.F32, held.up(rows), place, held.up(w), m, top_k, width, d_rows, d_w)
    base = back(rows, w, resid)
    scale = (np.abs(resid) + np.abs(w).sum(1, keepdims=True) * 8.0 + np.abs(w_step).sum(1, keepdims=True) * 8.0) * np.abs(dy)
    tol = 4 * (top_k + 2) * 2.0 ** -24 * scale.sum()  # two sums of at most 8 sigma rows on either side of the difference
    r2 = (rows + row_step).astype(np.float32)
    along = (d_rows.download().reshape(slots, width).astype(np.float64) * (r2.astype(np.float64) - rows)).sum()
    assert abs(((back(r2, w, resid) - base) * dy).sum() - along) <= tol
    w2 = (w + w_step).astype(np.float32)
    along = (d_w.download().reshape(m, top_k).astype(np.float64) * (w2.astype(np.float64) - w)).sum()
    # d_w's own dots: a rounding an addend
    extra = (width + 2) * 2.0 ** -24 * (np.abs(dy).sum(1) * 8.0 * np.abs(w_step).sum(1)).sum()
    assert abs(((back(rows, w2, resid) - base) * dy).sum() - along) <= tol + extra
    clean(gpu)


@DTYPES
def test_places_that_are_none(gpu, held, dtype):
    """A place past the rows raises and adds nothing; the host's word is passed over in silence."""
    m, top_k, width = 3, 2, 16
    rows, tok = np.ones((6, width), np.float32), np.full((m, width), 0.5, np.float32)
    place = np.array([0, 6, 0xFFFFFFFF, 1, 0x7FFFFFFF, 0xFFFFFFFF], U32)
    w = held.up(np.full(6, 2.0, np.float32))
    rd, td, pd = held.up(bits(rows, dtype)), held.up(bits(tok, dtype)), held.up(place)
    gpu.fault_clear()
    y = held.out(NUMPY[dtype], m * width)
    gpu.enqueue_expert_combine(rd, dtype, pd, w, td, m, top_k, width, y)
    assert np.array_equal(values(y.download(), dtype).reshape(m, width)[:, 0], [2.5, 2.5, 0.5])
    assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    gpu.fault_clear()
    d_rows, d_w = held.out(NUMPY[dtype], 6 * width), held.out(np.float32, 6)
    gpu.enqueue_expert_combine_grad(td, dtype, rd, pd, w, m, top_k, width, d_rows, d_w)
    assert np.array_equal(d_w.download(), [8.0, 0, 0, 8.0, 0, 0])
    words = d_rows.download().reshape(6, width)
    assert (values(words[:2], dtype) == 1.0).all() and (words[2:].view(np.uint8) == 0xEE).all()
    assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    gpu.fault_clear()


def test_infinities_stay_with_their_slots(gpu, held):
    r = Rows(held, bm.F32, 4, 8, 2, 32, 9, away=0.0)
    place = np.arange(8, dtype=U32)
    rows = np.ones((8, 32), np.float32)
    rows[2, 5], rows[4, 6] = np.inf, np.nan
    y = held.out(np.float32, 4 * 32)
    gpu.enqueue_expert_combine(held.up(rows), bm.F32, held.up(place), held.up(np.ones((4, 2), np.float32)), None, 4, 2, 32, y)
    got = y.download().reshape(4, 32)
    want = np.full((4, 32), 2.0)
    want[1, 5], want[2, 6] = np.inf, np.nan
    assert np.array_equal(got, want, equal_nan=True)
    assert r.m == 4


@pytest.mark.parametrize("m", (30, 1200))
def test_sort_and_back_captured_and_replayed(gpu, held, m):
    """Forward and backward as one graph, replayed over other picks and rows, with eager work between the replays."""
    rng = np.random.default_rng(10)
    n, top_k, width, dtype = 16, 4, 96, bm.BF16
    slots = m * top_k
    sel, x, dy, w = held.out(U32, slots), held.out(np.uint16, m * width), held.out(np.uint16, m * width), held.out(np.float32, slots)
    order, start, place = held.out(U32, slots), held.out(U32, n + 1), held.out(U32, slots)
    rows, d_rows = held.out(np.uint16, slots * width), held.out(np.uint16, slots * width)
    y, dx, d_w = held.out(np.uint16, m * width), held.out(np.uint16, m * width), held.out(np.float32, slots)
    work = held.out(U32, max(1, bm.expert_sort_work(slots, n)))
    outs = (order, start, place, rows, d_rows, y, dx, d_w)

    def enqueue():
        gpu.enqueue_expert_sort(sel, m, top_k, n, x, dtype, width, order, start, place, rows, work)
        gpu.enqueue_expert_combine(rows, dtype, place, w, x, m, top_k, width, y)
        gpu.enqueue_expert_combine_grad(dy, dtype, rows, place, w, m, top_k, width, d_rows, d_w)
        gpu.enqueue_expert_sort_grad(d_rows, dtype, place, m, top_k, width, dx)

    sel.upload(picks(rng, m, n, top_k))
    gpu.capture_begin()
    enqueue()
    graph = gpu.capture_end()
    try:
        for _ in range(4):
            sel.upload(picks(rng, m, n, top_k))
            x.upload(bits(normal_f32(rng, (m, width)), dtype))
            dy.upload(bits(normal_f32(rng, (m, width)), dtype))
            w.upload(normal_f32(rng, slots))
            for b in outs:
                b.fill_bytes(0xEE)
            gpu.graph_launch(graph)
            replayed = [b.download() for b in outs]
            for b in outs:
                b.fill_bytes(0xEE)
            enqueue()
            gpu.sync()
            for a, b in zip(replayed, outs):
                assert np.array_equal(a.view(np.uint8), b.download().view(np.uint8))
    finally:
        gpu.graph_destroy(graph)
    clean(gpu)
