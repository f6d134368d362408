"""GPU tests of every form that the products in 8-bit integers and their quantizer take, at sizes that lead to it: all forms of a product give the
same bits, so they are held to the rule's value, or to one another. The integer sums of the references are formed in f64, which
holds them exactly."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
from common import normal_f32
from rows_common import NAMES, NUMPY, TORCH, bits, codes_of, lines, padded, rounded, tables
from test_gpu_i8 import Held, clean, gpu, held, junk_padded, picks, quantize, some_matrix  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu
PTR = torch.Tensor.data_ptr


def value(q, s, w, ws):
    """The product's f32 value, from exact sums."""
    sums = (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)
    return (sums * s[:, None]).astype(np.float32) * ws[None, :]


# by the count of tiles: waves sharing k (tiles of 16 x 16, 16 x 32, 32 x 32), then tiles of 32 x 64, 64 x 64 (two rings), 64 x 128, 128 x 128, 256 x
# 256, 256 x 224; k of three lines and a piece, of half a line, of many lines and an odd number of values
SIZES = ((7, 4000, 272), (16, 8200, 272), (1, 9001, 1030), (20, 8300, 100), (90, 1200, 272), (250, 1000, 2056), (40, 9000, 272), (200, 1600, 272), (250, 2000, 1040), (700, 1100, 272), (700, 1100, 40), (650, 1300, 1111),
         (1600, 1400, 272), (1500, 1500, 144), (2050, 1600, 272), (2300, 2300, 272), (2301, 2299, 130), (4000, 4000, 272), (4001, 3999, 30), (4000, 3500, 272), (3990, 3490, 650))


@pytest.mark.parametrize("m,rows,k", SIZES)
def test_product_in_every_form(gpu, held, m, rows, k):
    rng = np.random.default_rng(m + rows + k)
    w, ws = some_matrix(rng, rows, k)
    q = rng.integers(-127, 128, (m, k), dtype=np.int16).astype(np.int8)
    s = rng.random(m).astype(np.float32)
    dtype = (bm.F32, bm.F16, bm.BF16)[k % 3]
    y = held.out(NUMPY[dtype], m * rows)
    gpu.enqueue_i8_gemm(held.up(junk_padded(w, k, rng)), held.up(ws), rows, k, held.up(padded(q, k)), held.up(s), m, y, dtype)
    got, want = y.download().reshape(m, rows), bits(value(q, s, w, ws), dtype)
    assert np.array_equal(got, want), f"{np.count_nonzero(got != want)} of {got.size} values differ"
    clean(gpu)


# by slots an expert and the count of tiles: 256 x 256, 128 x 128, 64 x 256, 64 x 128, 32 x 64 (two rings), 64 x 64 (two rings), waves sharing k; behind
# more than one reading of 256 bounds
@pytest.mark.parametrize("m,n,top_k,rows,k", ((1100, 2, 1, 300, 272), (900, 3, 2, 513, 40), (200, 64, 4, 2900, 48), (330, 90, 4, 3100, 144), (20, 300, 4, 70, 272), (200, 1000, 2, 40, 16),
                                              (999, 512, 8, 100, 48), (12, 1024, 3, 257, 272), (3000, 8, 1, 2000, 48), (1500, 8, 1, 3010, 144), (900, 8, 1, 4500, 48), (64, 128, 2, 700, 272), (50, 30, 4, 600, 272), (300, 9, 1, 333, 400),
                                              (700, 10, 1, 1500, 100), (40, 32, 4, 96, 400)))
@pytest.mark.parametrize("own", (False, True), ids=("shared", "own"))
def test_experts_product_in_every_form(gpu, held, own, m, n, top_k, rows, k):
    rng = np.random.default_rng(m + n + rows)
    ids = picks(rng, m, n, top_k)
    order, start, _ = tables(ids, n)
    n_slots, listed = m * top_k, int(start[-1])
    full = np.full(n_slots, 0x12345678, np.uint32)
    full[:listed] = order
    w, ws = some_matrix(rng, n * rows, k)
    cols = n_slots if own else m
    q = rng.integers(-127, 128, (cols, k), dtype=np.int16).astype(np.int8)
    s = rng.random(cols).astype(np.float32)
    y = held.out(np.float32, n_slots * rows)
    gpu.enqueue_i8_gemm_experts(held.up(junk_padded(w, k, rng)), held.up(ws), n, rows, k, held.up(padded(q, k)), held.up(s), None if own else held.up(full), held.up(start),
                                n_slots, 0 if own else top_k, y, bm.F32)
    got = y.download().reshape(n_slots, rows)
    col = np.arange(listed) if own else order // top_k
    for e in range(n):
        a, b = int(start[e]), int(start[e + 1])
        if b > a:
            want = value(q[col[a:b]], s[col[a:b]], w[e * rows:(e + 1) * rows], ws[e * rows:(e + 1) * rows])
            assert np.array_equal(got[a:b], want), f"expert {e}"
    assert (got[listed:].view(np.uint8) == 0xEE).all()
    clean(gpu)


@pytest.mark.parametrize("rows", (40, 300))
@pytest.mark.parametrize("own", (False, True), ids=("shared", "own"))
def test_tables_that_are_none_in_tiles(gpu, held, own, rows):
    """Runs outside the slots are skipped and raise, runs of nothing write nothing, an entry whose slot does not exist is NaN: of more slots than a
    wave's columns."""
    rng = np.random.default_rng(31 + rows)
    n, n_slots, top_k, k = 5, 150, 2, 272
    w, ws = some_matrix(rng, n * rows, k)
    cols = n_slots if own else n_slots // top_k
    q = rng.integers(-127, 128, (cols, k), dtype=np.int16).astype(np.int8)
    s = rng.random(cols).astype(np.float32)
    order = rng.permutation(n_slots).astype(np.uint32)
    wd, wsd, qd, sd = held.up(junk_padded(w, k, rng)), held.up(ws), held.up(padded(q, k)), held.up(s)
    gpu.fault_clear()
    for start, runs in (((0, 0, 0, 0, 0, 0), {}), ((7, 7, 7, 7, 7, 7), {}), ((0, 40, 30, 0xFFFFFFF0, 70, 150), {0: (0, 40), 4: (70, 150)}),
                        ((0, 70, 70, 71, 149, 151), {0: (0, 70), 2: (70, 71), 3: (71, 149)}), ((151, 152, 0xFFFFFFFF, 3, 3, 90), {4: (3, 90)})):
        y = held.out(np.float32, n_slots * rows)
        gpu.enqueue_i8_gemm_experts(wd, wsd, n, rows, k, qd, sd, None if own else held.up(order), held.up(np.array(start, np.uint32)), n_slots, 0 if own else top_k, y, bm.F32,
                                    n_cols=cols)
        got, done = y.download().reshape(n_slots, rows), np.zeros(n_slots, bool)
        for e, (a, b) in runs.items():
            col = np.arange(a, b) if own else order[a:b] // top_k
            assert np.array_equal(got[a:b], value(q[col], s[col], w[e * rows:(e + 1) * rows], ws[e * rows:(e + 1) * rows])), e
            done[a:b] = True
        assert (got[~done].view(np.uint32) == 0xEEEEEEEE).all()
        raised = gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
        assert raised == any(a > b or b > n_slots for a, b in zip(start, start[1:]))
        gpu.fault_clear()
    if own:
        return
    bad = order.copy()
    bad[[0, 9, 149]] = [n_slots, 0xFFFFFFFF, 0x80000000]
    y = held.out(np.float32, n_slots * rows)
    gpu.enqueue_i8_gemm_experts(wd, wsd, n, rows, k, qd, sd, held.up(bad), held.up(np.array((0, 40, 90, 91, 91, 150), np.uint32)), n_slots, top_k, y, bm.F32)
    got = y.download().reshape(n_slots, rows)
    assert np.isnan(got[[0, 9, 149]]).all() and np.isfinite(np.delete(got, [0, 9, 149], 0)).all()
    assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID
    gpu.fault_clear()


@pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)
@pytest.mark.parametrize("rows,k", ((40, 8), (40, 9), (100, 2048), (33, 2050), (20, 4090), (20, 4096), (20, 4101), (17, 8192), (50, 16384), (50, 16385), (4097, 77), (5000, 2048)))
def test_few_rows_in_one_call_are_the_two_calls(gpu, held, dtype, rows, k):
    rng = np.random.default_rng(rows + k)
    w, ws = some_matrix(rng, rows, k)
    wd, wsd, kp = held.up(junk_padded(w, k, rng)), held.up(ws), bm.i8_row_bytes(k)
    x = rounded(normal_f32(rng, (9, k)), dtype)
    codes, scales = codes_of(x)
    for m in range(1, 10):
        c1, s1 = quantize(gpu, held, x[:m], dtype, k)
        y1, y2 = held.out(NUMPY[dtype], m * rows), held.out(NUMPY[dtype], (m + 1) * rows, 0x77)
        c2, s2 = held.out(np.int8, (m + 1) * kp, 0x33), held.out(np.float32, m + 1, 0x44)
        gpu.enqueue_i8_gemm(wd, wsd, rows, k, c1, s1, m, y1, dtype)
        gpu.enqueue_i8_gemm_x(wd, wsd, rows, k, held.up(bits(x[:m], dtype)), dtype, m, c2, s2, y2, dtype)
        assert np.array_equal(c1.download().reshape(m, kp), padded(codes[:m], k)) and np.array_equal(s1.download(), scales[:m])
        assert np.array_equal(y1.download(), y2.download()[:m * rows]), m
        assert np.array_equal(c1.download(), c2.download()[:m * kp]) and np.array_equal(s1.download(), s2.download()[:m])
        # the row behind the last is left as it was
        assert (y2.download()[m * rows:].view(np.uint8) == 0x77).all() and (c2.download()[m * kp:] == 0x33).all()
        assert (s2.download()[m:].view(np.uint8) == 0x44).all()
    clean(gpu)


@pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)
@pytest.mark.parametrize("m,k", ((3, 3), (2100, 5), (30, 1020), (30, 2050), (2100, 2050), (2060, 4096), (30, 4099), (2100, 4099), (30, 8191), (2060, 8192), (5, 8193), (3, 40000)))
def test_quantizer_in_every_form(gpu, held, dtype, m, k):
    rng = np.random.default_rng(m + k)
    x = rounded(normal_f32(rng, (m, k)), dtype)
    q, s = codes_of(x)
    codes, scales = quantize(gpu, held, x, dtype, k, ld=k + 1)
    assert np.array_equal(scales.download(), s)
    assert np.array_equal(codes.download().reshape(m, -1), padded(q, k))
    # the gate rule's values: rows by themselves (a form for few of them) and all together
    g, u = x, rounded(normal_f32(rng, (m, k)), dtype)
    gd, ud, kp = held.up(bits(g, dtype)), held.up(bits(u, dtype)), bm.i8_row_bytes(k)
    c1, s1, c2, s2 = held.out(np.int8, m * kp), held.out(np.float32, m), held.out(np.int8, 2 * kp), held.out(np.float32, 2)
    gpu.enqueue_i8_swiglu_quantize(gd, ud, dtype, m, k, c1, s1)
    gpu.enqueue_i8_swiglu_quantize(held.up(bits(g[-2:], dtype)), held.up(bits(u[-2:], dtype)), dtype, 2, k, c2, s2)
    assert np.array_equal(c1.download()[-2 * kp:], c2.download()) and np.array_equal(s1.download()[-2:], s2.download())
    silu = g[-2:] / (1 + np.exp(-g[-2:])) * u[-2:]
    # a code's value is within half a step of the scale, and two f32 roundings and an exponential's few ulps of the gate's
    step = s2.download().astype(np.float64)[:, None]
    assert (np.abs(c2.download().reshape(2, kp)[:, :k] * step - silu) <= step * (0.5 + 127 * 2.0 ** -20)).all()
    clean(gpu)


def test_offsets_past_32_bits(gpu):
    """A matrix of 4.3 GB as rows, as columns, as gathered columns and as an expert's rows: its last rows against sums on the host."""
    k, n = 131072, 32800
    torch.manual_seed(3)
    big = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda")
    few = torch.randint(-127, 128, (40, k), dtype=torch.int8, device="cuda")
    big_s, few_s = torch.rand(n, device="cuda"), torch.rand(40, device="cuda")
    at = torch.tensor([0, 5, 16383, 16384, n - 33, n - 2, n - 1])
    sums = (big[at.cuda()].cpu().double() @ few.cpu().double().t()).float()
    b, f = big_s.cpu()[at][:, None], few_s.cpu()[None]
    as_rows, as_columns = (sums * f) * b, (sums * b) * f
    for m in (1, 40):
        y = torch.zeros(m, n, device="cuda")
        torch.cuda.synchronize()
        gpu.enqueue_i8_gemm(PTR(big), PTR(big_s), n, k, PTR(few), PTR(few_s), m, PTR(y), bm.F32)
        gpu.sync()
        assert torch.equal(y.cpu()[:, at], as_rows[:, :m].t()), m
    y = torch.zeros(n, 40, device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_i8_gemm(PTR(few), PTR(few_s), 40, k, PTR(big), PTR(big_s), n, PTR(y), bm.F32)
    gpu.sync()
    assert torch.equal(y.cpu()[at], as_columns)
    # the columns behind an order, of one expert's 40 slots: offsets of gathered columns past 32 bits
    order = torch.cat((at, torch.arange(33))).int().cuda()
    start, y = torch.tensor([0, 40], dtype=torch.int32, device="cuda"), torch.zeros(40, 40, device="cuda")
    torch.cuda.synchronize()
    slots = n  # every column's slot exists; one expert's run lists forty of them
    table = torch.zeros(slots, dtype=torch.int32, device="cuda")
    table[:40] = order
    y = torch.zeros(slots, 40, device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_i8_gemm_experts(PTR(few), PTR(few_s), 1, 40, k, PTR(big), PTR(big_s), PTR(table), PTR(start), slots, 1, PTR(y), bm.F32, n_cols=n)
    gpu.sync()
    assert torch.equal(y.cpu()[:7], as_columns) and not y[40:].any()
    # two experts of 16400 rows, the second's past 32 bits
    y = torch.zeros(40, n // 2, device="cuda")
    start = torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_i8_gemm_experts(PTR(big), PTR(big_s), 2, n // 2, k, PTR(few), PTR(few_s), None, PTR(start), 40, 0, PTR(y), bm.F32)
    gpu.sync()
    inside = at[4:] - n // 2
    assert torch.equal(y.cpu()[20:, inside], as_rows[4:, 20:].t())
    clean(gpu)


def test_two_contexts_at_once(gpu):
    """Two contexts, each on a stream of its own with the buffers of its own call, and the same weights: neither waits for nor disturbs the other."""
    rng = np.random.default_rng(21)
    rows, k, m = 700, 1000, 300
    w, ws = some_matrix(rng, rows, k)
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = [bm.Gpu(0, stream=s.cuda_stream) for s in streams]
    try:
        wt, wst = torch.from_numpy(junk_padded(w, k, rng)).cuda(), torch.from_numpy(ws).cuda()
        xs = [torch.from_numpy(normal_f32(rng, (m, k))).cuda() for _ in range(2)]
        outs = [(torch.zeros(m, bm.i8_row_bytes(k), dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda"), torch.zeros(m, rows, device="cuda")) for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(20):
            for c, x, (codes, scales, y) in zip(contexts, xs, outs):
                c.enqueue_i8_gemm_x(PTR(wt), PTR(wst), rows, k, PTR(x), bm.F32, m, PTR(codes), PTR(scales), PTR(y), bm.F32)
        torch.cuda.synchronize()
        for x, (_, _, y) in zip(xs, outs):
            q, s = codes_of(x.cpu().numpy())
            assert np.array_equal(y.cpu().numpy(), value(q, s, w, ws))
    finally:
        for c in contexts:
            c.close()


@pytest.mark.parametrize("m", (1, 6, 40, 700))
def test_a_product_captured_and_replayed(gpu, held, m):
    """Two products behind one another as one graph, replayed over other rows with eager work between the replays."""
    rng = np.random.default_rng(41 + m)
    hidden, rows, dtype = 512, 1100, bm.BF16
    w1, ws1 = some_matrix(rng, rows, hidden)
    w2, ws2 = some_matrix(rng, hidden, rows)
    d1, s1, d2, s2 = held.up(w1), held.up(ws1), held.up(junk_padded(w2, rows, rng)), held.up(ws2)
    x, y, z = held.out(np.uint16, m * hidden), held.out(np.uint16, m * rows), held.out(np.uint16, m * hidden)
    codes, scales = held.out(np.int8, m * bm.i8_row_bytes(rows)), held.out(np.float32, m)

    def enqueue():
        gpu.enqueue_i8_gemm_x(d1, s1, rows, hidden, x, dtype, m, codes, scales, y, dtype)
        gpu.enqueue_i8_gemm_x(d2, s2, hidden, rows, y, dtype, m, codes, scales, z, dtype)

    x.upload(bits(normal_f32(rng, (m, hidden)), dtype))
    gpu.capture_begin()
    enqueue()
    graph = gpu.capture_end()
    try:
        for _ in range(3):
            xf = rounded(normal_f32(rng, (m, hidden)), dtype)
            x.upload(bits(xf, dtype))
            for b in (y, z, codes, scales):
                b.fill_bytes(0xEE)
            gpu.graph_launch(graph)
            replayed = [b.download() for b in (y, z, codes, scales)]
            q, s = codes_of(xf)
            assert np.array_equal(replayed[0].reshape(m, rows), bits(value(q, s, w1, ws1), dtype))
            for b in (y, z, codes, scales):
                b.fill_bytes(0x11)
            enqueue()
            gpu.sync()
            for a, b in zip(replayed, (y, z, codes, scales)):
                assert np.array_equal(a.view(np.uint8), b.download().view(np.uint8))
    finally:
        gpu.graph_destroy(graph)
    clean(gpu)


@pytest.mark.parametrize("n,bad", ((60, 59), (100, 70), (300, 64), (300, 255), (300, 299), (1024, 900)))
def test_a_run_that_is_none_far_behind_the_first_raises(gpu, held, n, bad):
    """Wherever in the table: the runs in front of it and behind it are computed, and the fault is there."""
    rng = np.random.default_rng(n + bad)
    n_slots, rows, k = 700, 130, 48
    w, ws = some_matrix(rng, n * rows, k)
    q = rng.integers(-127, 128, (n_slots, k), dtype=np.int16).astype(np.int8)
    s = rng.random(n_slots).astype(np.float32)
    start = np.linspace(0, n_slots, n + 1).astype(np.uint32)
    wd, wsd, qd, sd = held.up(w), held.up(ws), held.up(q), held.up(s)
    for end in (None, n_slots + 1, 0xFFFFFFFF):
        table = start.copy()
        if end is not None:
            table[bad + 1] = end  # the run `bad` passes the slots, and the one behind it runs backwards
        gpu.fault_clear()
        y = held.out(np.float32, n_slots * rows)
        gpu.enqueue_i8_gemm_experts(wd, wsd, n, rows, k, qd, sd, None, held.up(table), n_slots, 0, y, bm.F32)
        got, done = y.download().reshape(n_slots, rows), np.zeros(n_slots, bool)
        for e in range(n):
            a, b = int(table[e]), int(table[e + 1])
            if a <= b <= n_slots:
                assert np.array_equal(got[a:b], value(q[a:b], s[a:b], w[e * rows:(e + 1) * rows], ws[e * rows:(e + 1) * rows])), e
                done[a:b] = True
        assert (got[~done].view(np.uint32) == 0xEEEEEEEE).all()
        assert (gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID) == (end is not None)
        gpu.fault_clear()


def needs_memory(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"{gigabytes} GiB of the card's memory are not free")


def test_the_most_rows_of_the_longest_form(gpu):
    """2^22 rows past 8192 values, a workgroup of 1024 threads each: 2^32 threads. Rows of zeros, some others spread among them."""
    needs_memory(110)
    m, k = 1 << 22, 8193
    kp = bm.i8_row_bytes(k)
    at = torch.tensor([0, 1, (1 << 20) - 1, 1 << 20, (1 << 21) + 7, 3 << 20, m - 2, m - 1])
    torch.manual_seed(5)
    some = torch.randn(at.numel(), k).bfloat16()
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[at.cuda()] = some.cuda()
    codes, scales = torch.empty(m, kp, dtype=torch.int8, device="cuda").fill_(0x55), torch.full((m,), -1.0, device="cuda")
    q, s = codes_of(some.float().numpy())
    live = torch.tensor([m - 1], dtype=torch.int32, device="cuda")
    try:
        for n, word in ((m - 1, PTR(live)), (m, None)):
            torch.cuda.synchronize()
            gpu.enqueue_i8_quantize(PTR(x), bm.BF16, m, k, PTR(codes), PTR(scales), live=word)
            gpu.sync()
            if n < m:  # the row behind the last is left as it was
                assert (codes[n:].cpu() == 0x55).all() and scales[n].item() == -1.0
            there = at[at < n]
            assert np.array_equal(codes[there.cuda()].cpu().numpy(), padded(q[:there.numel()], k))
            want = torch.zeros(n)
            want[there] = torch.from_numpy(s)[:there.numel()]
            assert torch.equal(scales[:n].cpu(), want)
        codes[at.cuda()] = 0
        for part in codes.view(torch.int64).split(1 << 19):
            assert not part.any().item()
        clean(gpu)
    finally:
        del x, codes
        torch.cuda.empty_cache()


def test_the_most_rows_an_expert(gpu):
    """Experts of 2^22 rows each: more than 2^32 threads of tiles, counted by the most that the runs may make."""
    needs_memory(70)
    n, rows, k = 600, 1 << 22, 16
    torch.manual_seed(6)
    w, ws = torch.empty(n * rows, k, dtype=torch.int8, device="cuda"), torch.empty(n * rows, device="cuda")
    for part, scales in zip(w.split(1 << 28), ws.split(1 << 28)):
        part.random_(-127, 128)
        scales.uniform_()
    q, s = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda"), torch.rand(n, device="cuda")
    # a slot an expert, but for one with none and its neighbour with two
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    start[8] = 7
    y = torch.empty(n, rows, dtype=torch.bfloat16, device="cuda").fill_(float("nan"))
    try:
        torch.cuda.synchronize()
        gpu.enqueue_i8_gemm_experts(PTR(w), PTR(ws), n, rows, k, PTR(q), PTR(s), None, PTR(start), n, 0, PTR(y), bm.BF16)
        gpu.sync()
        for e in range(n):
            a, b = int(start[e]), int(start[e + 1])
            sums = q[a:b].float() @ w[e * rows:(e + 1) * rows].float().t()  # exact: below 2^24
            assert torch.equal(y[a:b], (sums * s[a:b, None] * ws[e * rows:(e + 1) * rows]).bfloat16()), e
        clean(gpu)
    finally:
        del w, ws, y, part, scales
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)
@pytest.mark.parametrize("m,k", ((2100, 5), (300, 500), (301, 770), (30, 2050), (2100, 2050), (100, 1500), (2061, 4096), (2100, 4099), (40, 8191), (2060, 8192), (9, 8193), (5, 40000)))
def test_the_gate_rules_values_of_every_row(gpu, held, dtype, m, k):
    """Codes and scales of every row against silu(g) u in 64 bits, in every form: the exponential, the divide and the products are off by 64 x 2^-24
    at most, a scale by that and its own rounding, a code by half a step and twice that of at most 127."""
    rng = np.random.default_rng(3 * m + k)
    scale = np.exp(normal_f32(rng, (m, 1)))  # rows that no other row's scale fits
    g, u = rounded(normal_f32(rng, (m, k)), dtype), rounded(normal_f32(rng, (m, k)) * scale, dtype)
    kp, ld = bm.i8_row_bytes(k), k + 1
    codes, scales = held.out(np.int8, (m + 1) * kp, 0x55), held.out(np.float32, m + 1)
    gpu.enqueue_i8_swiglu_quantize(held.up(lines(g, dtype, ld, np.nan)), held.up(lines(u, dtype, ld, np.nan)), dtype, m, k, codes, scales, ld=ld)
    h = g / (1 + np.exp(-g)) * u
    step = np.abs(h).max(axis=1) / 127
    got, s = codes.download().reshape(m + 1, kp), scales.download()
    tol = 64 * 2.0 ** -24
    assert np.allclose(s[:m], step, rtol=tol + 2.0 ** -23, atol=0)
    assert (np.abs(got[:m, :k] - h / step[:, None]) <= 0.5 + 127 * (2 * tol + 2.0 ** -22)).all()
    assert (np.abs(got[:m].astype(int)).max(axis=1) == 127).all() and not got[:m, k:].any()
    assert (got[m] == 0x55).all() and s[m:].view(np.uint32)[0] == 0xEEEEEEEE
    clean(gpu)
