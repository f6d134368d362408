"""GPU tests of every form that the products in microscaled 4-bit floating point take, at sizes that lead to it (which size leads to which is held by
test_mx4_forms_cpu.py, without a device): one line of k to thirteen, whole last lines and ragged ones, rows and columns that are no multiples of a tile's. The
references are formed in f64, which holds the codes' products and their sums under these scales exactly."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
import mx4_common as mx
from rows_common import HALF_STEP, NAMES, TORCH, tables
from test_gpu_mx4 import clean, gpu, picks  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
PTR = torch.Tensor.data_ptr

# lines of 256 values: 1, 1, 2, 3, 4, 6, 9, 10, 13; blocks of the last one: 2, 8, 2, 1, 8, 1, 1, 8, 6
KS = (40, 256, 300, 520, 1024, 1300, 2080, 2560, 3250)
# (columns, rows, waves, buffers) of a form: sizes (columns, rows) that take it
ONE = {(16, 16, 8, 4): ((40, 90), (1, 4001)), (16, 32, 3, 4): ((9, 8300), (60, 1700)), (32, 32, 4, 4): ((20, 8300), (100, 2000)), (32, 64, 2, 2): ((200, 1600), (33, 9001)),
       (64, 64, 4, 2): ((700, 1900), (1500, 1111)), (128, 128, 4, 2): ((640, 12800),), (256, 128, 8, 2): ((2300, 2299),), (256, 256, 8, 2): ((4000, 4000),)}
# sizes (tokens, experts, top_k, rows an expert)
EXPERTS = {(16, 32, 3, 4): ((5, 6, 3, 200), (40, 8, 2, 300)), (32, 64, 2, 2): ((250, 128, 2, 700), (400, 8, 2, 700), (90, 300, 2, 1000)),
           (64, 64, 4, 2): ((640, 32, 2, 2500), (600, 8, 2, 2000)), (128, 128, 4, 2): ((1500, 32, 2, 1500), (800, 4, 1, 4800)),
           (256, 256, 8, 2): ((1100, 2, 1, 4000), (3000, 8, 1, 1500))}


def rows_of(gen, n, k, zeros):
    """Codes and scales as a device holds them: anything behind the last block's scale, and behind the k-th code zeros or anything."""
    w = torch.randint(0, 256, (n, mx.row_bytes(k)), dtype=torch.uint8, device="cuda", generator=gen)
    if zeros:
        if k % 2:
            w[:, k // 2] &= 15
        w[:, (k + 1) // 2:] = 0
    s = torch.randint(117, 126, (n, mx.row_scales(k)), dtype=torch.uint8, device="cuda", generator=gen)
    s[:, -(-k // 32):] = 255
    return w, s


def values_of(w, s, k):
    level = torch.tensor(mx.LEVELS, device="cuda")
    level = torch.cat([level, -level])
    v = torch.stack([level[(w & 15).long()], level[(w >> 4).long()]], 2).view(w.shape[0], -1, 32)
    return (v * torch.exp2(s[:, :v.shape[1]].double() - 127)[:, :, None]).view(w.shape[0], -1)[:, :k]


def assert_near(y, dtype, x, v, what=""):
    exact = x @ v.t().contiguous()
    bound = (-(-x.shape[1] // 32) + 8) * mx.STEP * (x.abs() @ v.abs().t().contiguous())  # mx4_common.product_bound
    off = HALF_STEP[dtype] * (exact.abs() + bound) + bound + (2.0 ** -25 if dtype == bm.F16 else 0.0)
    assert ((y.double() - exact).abs() <= off).all(), what


@pytest.mark.parametrize("k", KS)
@pytest.mark.parametrize("m,rows", [s for sizes in ONE.values() for s in sizes])
def test_one_matrix(gpu, m, rows, k):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m + rows + k)
    w, q = rows_of(gen, rows, k, False), rows_of(gen, m, k, True)
    dtype = (bm.F32, bm.F16, bm.BF16)[(KS.index(k) + m) % 3]
    y = torch.full((m, rows + 1), 7.0, dtype=TORCH[dtype], device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_mx4_gemm(PTR(w[0]), PTR(w[1]), rows, k, PTR(q[0]), PTR(q[1]), m, PTR(y), dtype, ld_y=rows + 1)
    gpu.sync()
    assert_near(y[:, :rows], dtype, values_of(*q, k), values_of(*w, k))
    assert (y[:, rows] == 7.0).all()
    clean(gpu)


@pytest.mark.parametrize("k", KS[::2])
@pytest.mark.parametrize("own", (False, True), ids=("shared", "own"))
@pytest.mark.parametrize("m,n,top_k,rows", [s for sizes in EXPERTS.values() for s in sizes])
def test_experts(gpu, m, n, top_k, rows, own, k):
    rng = np.random.default_rng(m + n + rows + k)
    order, start, _ = tables(picks(rng, m, n, top_k, away=0.1), n)
    n_slots, listed = m * top_k, order.size
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m + n + rows + k)
    w, q = rows_of(gen, n * rows, k, False), rows_of(gen, n_slots if own else m, k, True)
    dtype = (bm.BF16, bm.F32, bm.F16)[(KS.index(k) // 2 + m) % 3]
    full = np.full(n_slots, 0x12345678, np.uint32)
    full[:listed] = order
    table, bounds = torch.from_numpy(full.view(np.int32)).cuda(), torch.from_numpy(start.view(np.int32)).cuda()
    col = torch.arange(listed, device="cuda") if own else torch.from_numpy(order.astype(np.int64)).cuda() // top_k
    y = torch.full((n_slots, rows), 7.0, dtype=TORCH[dtype], device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_mx4_gemm_experts(PTR(w[0]), PTR(w[1]), n, rows, k, PTR(q[0]), PTR(q[1]), None if own else PTR(table), PTR(bounds), n_slots, 0 if own else top_k, PTR(y), dtype)
    gpu.sync()
    x = values_of(*q, k)
    for e in range(n):
        a, b = int(start[e]), int(start[e + 1])
        if b > a:
            of = slice(e * rows, (e + 1) * rows)
            assert_near(y[a:b], dtype, x[col[a:b]], values_of(w[0][of], w[1][of], k), f"expert {e}")
    assert (y[listed:] == 7.0).all()
    clean(gpu)


@pytest.mark.parametrize("form", EXPERTS, ids=lambda f: "x".join(map(str, f)))
def test_tables_that_are_none_in_every_form(gpu, form):
    """A run past the slots and one that runs backwards are skipped and raised, an entry that names no slot gets NaN, in every form."""
    m, n, top_k, rows = EXPERTS[form][0]
    k, n_slots = 300, m * top_k
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    w, q = rows_of(gen, n * rows, k, False), rows_of(gen, m, k, True)
    table = torch.randperm(n_slots, device="cuda", generator=gen).int()
    for kind in ("past", "back", "entry"):
        start = torch.linspace(0, n_slots, n + 1, device="cuda").round().int()
        order = table.clone()
        ran = torch.ones(n_slots, dtype=torch.bool, device="cuda")
        nan = torch.zeros_like(ran)
        if kind == "past":
            ran[int(start[n - 1]):] = False
            start[n] = n_slots + 5
        elif kind == "back":
            ran[int(start[0]):int(start[1])] = False
            start[0] = 0x7FFFFFF0
        else:
            order[n_slots - 1], order[0] = n_slots, -1
            nan[0] = nan[n_slots - 1] = True
        y = torch.full((n_slots, rows), 7.0, device="cuda")
        gpu.fault_clear()
        torch.cuda.synchronize()
        gpu.enqueue_mx4_gemm_experts(PTR(w[0]), PTR(w[1]), n, rows, k, PTR(q[0]), PTR(q[1]), PTR(order), PTR(start), n_slots, top_k, PTR(y), bm.F32)
        gpu.sync()
        assert gpu.fault()[0] & 0xFF == bm.SITE_EXPERT_ID, kind
        assert (y[~ran] == 7.0).all() and torch.isnan(y[nan]).all() and torch.isfinite(y[~nan]).all(), kind
        j = int(start[1]) if kind != "past" else 0
        e = 1 if kind != "past" else 0
        if int(start[e + 1]) > j and not bool(nan[j]):
            of = slice(e * rows, (e + 1) * rows)
            assert_near(y[j:j + 1], bm.F32, values_of(*q, k)[order[j:j + 1].long() // top_k], values_of(w[0][of], w[1][of], k), kind)
    gpu.fault_clear()


# (form, columns, experts, rows): columns past 2^31 bytes, and the most that 32 bits hold; the last one's are past them
FAR = (((32, 64, 2, 2), 38000, 1, 40), ((64, 64, 4, 2), 45000, 1, 40), ((128, 128, 4, 2), 65535, 200, 100), ((256, 256, 8, 2), 65535, 1, 300), ((16, 32, 3, 4), 65536, 3, 50))


def test_gathered_columns_far_into_the_tiles_reach(gpu):
    """Columns of up to 4.3 GB behind an order, in every form that such a table takes; and one column more, which goes by whole addresses."""
    k = 131072
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    q, s = rows_of(gen, 65536, k, True)
    for form, cols, n, rows in FAR:
        assert bm.mx4_gemm_form(rows, k, cols, n, cols, 1) == form
        listed = torch.tensor([cols - 1, 0, 32767, 32768, 32769, cols - 2] + list(range(cols - 60, cols - 20)), device="cuda")
        table = torch.full((cols,), 0x12345678, dtype=torch.int32, device="cuda")
        table[:listed.numel()] = listed.int()
        w, ws = rows_of(gen, n * rows, k, False)
        start = torch.full((n + 1,), 4, dtype=torch.int32, device="cuda")  # the first expert's four, and the last one's others
        start[0], start[n] = 0, listed.numel()
        y = torch.full((cols, rows), 7.0, device="cuda")
        torch.cuda.synchronize()
        gpu.enqueue_mx4_gemm_experts(PTR(w), PTR(ws), n, rows, k, PTR(q), PTR(s), PTR(table), PTR(start), cols, 1, PTR(y), bm.F32)
        gpu.sync()
        for e in {0, n - 1}:
            at = torch.arange(int(start[e]), int(start[e + 1]), device="cuda")
            of, col = slice(e * rows, (e + 1) * rows), listed[at]
            assert_near(y[at], bm.F32, values_of(q[col], s[col], k), values_of(w[of], ws[of], k), form)
        assert (y[listed.numel():] == 7.0).all()
    clean(gpu)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m,rows,k", ((40, 90, 2000), (700, 1900, 2000), (2300, 2299, 1000)))
def test_captured_and_replayed_while_another_context_works(gpu, m, rows, k):
    """The same call twice gives the same bits, eager, replayed, and beside a second context on a stream of its own."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    w, x = rows_of(gen, rows, k, False), torch.randn(m, k, device="cuda", generator=gen)
    other = bm.Gpu(0)
    buffers = [(torch.zeros(m, mx.row_bytes(k), dtype=torch.uint8, device="cuda"), torch.zeros(m, mx.row_scales(k), dtype=torch.uint8, device="cuda"), torch.zeros(m, rows, device="cuda"))
               for _ in range(3)]
    torch.cuda.synchronize()

    def call(g, b):
        g.enqueue_mx4_gemm_x(PTR(w[0]), PTR(w[1]), rows, k, PTR(x), bm.F32, m, PTR(b[0]), PTR(b[1]), PTR(b[2]), bm.F32)

    call(gpu, buffers[0])
    gpu.sync()
    gpu.capture_begin()
    call(gpu, buffers[1])
    graph = gpu.capture_end()
    try:
        for turn in range(3):
            for b in buffers[1:]:
                b[2].fill_(7.0)
            torch.cuda.synchronize()
            gpu.graph_launch(graph)
            for _ in range(3):
                call(other, buffers[2])
            gpu.sync()
            other.sync()
            for b in buffers[1:]:
                assert all(torch.equal(p, q) for p, q in zip(b, buffers[0])), turn
    finally:
        gpu.graph_destroy(graph)
        other.close()
    v = values_of(*w, k)
    assert_near(buffers[0][2], bm.F32, values_of(*buffers[0][:2], k), v)
    clean(gpu)


@pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)
@pytest.mark.parametrize("m,rows,k", ((1, 5000, 2048), (2, 5000, 8192), (3, 700, 4096), (4, 300, 4090), (8, 4500, 2048), (8, 64, 2049), (5, 64, 2049), (1, 40, 16384), (1, 40, 16390), (1, 7, 7),
                                      (9, 300, 1024), (16, 8192, 2048), (16, 4500, 2041), (16, 100, 2049), (12, 64, 40), (17, 300, 1024), (32, 8192, 1019), (32, 64, 1025), (31, 5000, 520), (24, 33, 8),
                                      (33, 64, 512), (8, 100, 4096), (8, 100, 4100), (4, 64, 8190), (3, 4200, 4097), (2, 40, 16384), (1, 40, 32768), (1, 40, 32770), (1, 8193, 100), (32, 8193, 512)))
def test_few_rows_at_either_end_of_one_launch(gpu, dtype, m, rows, k):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m + k)
    w, x = rows_of(gen, rows, k, False), (torch.randn(m, k + 3, device="cuda", generator=gen) * 3).to(TORCH[dtype])
    codes, scales = torch.full((m + 1, mx.row_bytes(k)), 0x55, dtype=torch.uint8, device="cuda"), torch.full((m + 1, mx.row_scales(k)), 0x55, dtype=torch.uint8, device="cuda")
    y = torch.full((m + 1, rows), 7.0, dtype=TORCH[dtype], device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_mx4_gemm_x(PTR(w[0]), PTR(w[1]), rows, k, PTR(x), dtype, m, PTR(codes), PTR(scales), PTR(y), dtype, ld_x=k + 3)
    gpu.sync()
    words, padded = mx.pack(*mx.encode(x[:, :k].double().cpu().numpy()), k)
    assert np.array_equal(codes[:m].cpu().numpy(), words) and np.array_equal(scales[:m].cpu().numpy(), padded)
    assert (codes[m] == 0x55).all() and (scales[m] == 0x55).all() and (y[m] == 7.0).all()
    assert_near(y[:m], dtype, values_of(codes[:m], scales[:m], k), values_of(*w, k))
    clean(gpu)


def test_a_value_that_is_not_finite_among_few_rows(gpu):
    m, rows, k = 3, 100, 700
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    w, x = rows_of(gen, rows, k, False), torch.randn(m, k, device="cuda", generator=gen)
    x[1, 333] = float("inf")
    codes, scales = torch.zeros(m, mx.row_bytes(k), dtype=torch.uint8, device="cuda"), torch.zeros(m, mx.row_scales(k), dtype=torch.uint8, device="cuda")
    y = torch.zeros(m, rows, device="cuda")
    gpu.fault_clear()
    torch.cuda.synchronize()
    gpu.enqueue_mx4_gemm_x(PTR(w[0]), PTR(w[1]), rows, k, PTR(x), bm.F32, m, PTR(codes), PTR(scales), PTR(y), bm.F32)
    gpu.sync()
    words, padded = mx.pack(*mx.encode(x.double().cpu().numpy()), k)
    assert np.array_equal(codes.cpu().numpy(), words) and np.array_equal(scales.cpu().numpy(), padded)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()
    assert gpu.fault()[0] & 0xFF == bm.SITE_QUANT_COLUMN
    gpu.fault_clear()


def needs_memory(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"{gigabytes} GiB of the card's memory are not free")


def test_the_most_rows_there_and_back(gpu):
    """2^22 rows of 8192 values, a wave every 512 of them: 2^32 threads. Rows of zeros, some others spread among them; and back into the same rows."""
    needs_memory(100)
    m, k = 1 << 22, 8192
    at = torch.tensor([0, 1, (1 << 20) - 1, 1 << 20, (1 << 21) + 7, 3 << 20, m - 2, m - 1])
    torch.manual_seed(5)
    some = torch.randn(at.numel(), k).bfloat16()
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[at.cuda()] = some.cuda()
    codes, scales = torch.full((m, k // 2), 0x55, dtype=torch.uint8, device="cuda"), torch.full((m, k // 32), 0x55, dtype=torch.uint8, device="cuda")
    q, b = mx.encode(some.double().numpy())
    words, padded = mx.pack(q, b, k)
    live = torch.tensor([m - 1], dtype=torch.int32, device="cuda")
    try:
        for n, word in ((m - 1, PTR(live)), (m, None)):
            torch.cuda.synchronize()
            gpu.enqueue_mx4_quantize(PTR(x), bm.BF16, m, k, PTR(codes), PTR(scales), live=word)
            gpu.sync()
            if n < m:
                assert (codes[n:] == 0x55).all() and (scales[n:] == 0x55).all()
            there = at[at < n]
            assert np.array_equal(codes[there.cuda()].cpu().numpy(), words[:there.numel()]) and np.array_equal(scales[there.cuda()].cpu().numpy(), padded[:there.numel()])
        gpu.enqueue_mx4_dequantize(PTR(codes), PTR(scales), m, k, PTR(x), bm.BF16)
        gpu.sync()
        assert np.array_equal(x[at.cuda()].double().cpu().numpy(), mx.decode(q, b, k))
        for held in (codes, scales, x):
            held[at.cuda()] = 0
            for part in held.view(torch.int64).split(1 << 19):
                assert not part.any().item()
        clean(gpu)
    finally:
        del x, codes, scales, held
        torch.cuda.empty_cache()


def test_the_most_rows_an_expert(gpu):
    """Experts of 2^22 rows each: more than 2^32 threads of tiles, counted by the most that the runs may make."""
    needs_memory(110)
    n, rows, k = 600, 1 << 22, 16
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    w, ws = torch.empty(n * rows, 16, dtype=torch.uint8, device="cuda"), torch.full((n * rows, 16), 255, dtype=torch.uint8, device="cuda")
    for part in w.split(1 << 28):
        part.random_(0, 256, generator=gen)
    for part in ws.split(1 << 28):
        part[:, 0].random_(117, 126, generator=gen)
    q = rows_of(gen, n, k, True)
    # a slot an expert, but for one with none and its neighbour with two
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    start[8] = 7
    y = torch.empty(n, rows, dtype=torch.bfloat16, device="cuda").fill_(float("nan"))
    try:
        torch.cuda.synchronize()
        gpu.enqueue_mx4_gemm_experts(PTR(w), PTR(ws), n, rows, k, PTR(q[0]), PTR(q[1]), None, PTR(start), n, 0, PTR(y), bm.BF16)
        gpu.sync()
        x = values_of(*q, k)
        for e in (0, 1, 6, 7, 8, 9, 300, n - 2, n - 1):
            a, b = int(start[e]), int(start[e + 1])
            for r in (slice(0, 5000), slice(rows - 5000, rows)):
                assert_near(y[a:b, r], bm.BF16, x[a:b], values_of(w[e * rows:(e + 1) * rows][r], ws[e * rows:(e + 1) * rows][r], k), e)
        assert torch.isfinite(y).all()
        clean(gpu)
    finally:
        del w, ws, y, part
        torch.cuda.empty_cache()
