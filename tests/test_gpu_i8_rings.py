"""GPU tests of the 8-bit products' forms over rows long enough that their rings of LDS buffers go round: nine to thirteen steps of 128 bytes,
an odd and an even number, last steps of one piece to eight. (Which form a size takes is held by test_i8_forms_cpu.py, without a device.)
Sums of the references are formed in f64, which holds them exactly."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
from rows_common import TORCH, tables
from test_gpu_i8 import clean, gpu, picks  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
PTR = torch.Tensor.data_ptr

KS = (1040, 1170, 1300, 1500, 1650)
# (columns, rows, waves, buffers) of a form: a size (columns, rows) that takes it with each of KS
ONE = {(16, 16, 8, 4): (40, 90), (16, 32, 4, 4): (20, 4000), (16, 32, 3, 4): (9, 8300), (32, 32, 4, 4): (20, 8300), (32, 64, 2, 4): (200, 1600),
       (64, 64, 4, 4): (700, 1100), (64, 64, 4, 2): (1500, 1500), (64, 128, 4, 2): (1600, 2000), (128, 128, 4, 2): (2300, 2299),
       (256, 224, 8, 2): (4000, 3500), (256, 256, 8, 2): (4000, 4000)}
# sizes (tokens, experts, top_k, rows an expert)
EXPERTS = {(16, 32, 3, 4): ((5, 6, 3, 200),), (32, 32, 4, 4): ((40, 32, 4, 96),), (32, 64, 2, 4): ((80, 16, 2, 700),), (64, 64, 4, 4): ((400, 8, 2, 700),),
           (64, 64, 4, 2): ((400, 8, 2, 2000),), (256, 256, 8, 2): ((1100, 2, 1, 4000),), (128, 128, 4, 2): ((800, 4, 1, 4800),),
           # rows of eight tiles and more, and of fewer, whose groups of tiles stay on a die
           (64, 256, 4, 2): ((960, 16, 2, 1800), (640, 64, 2, 900)), (64, 128, 4, 2): ((640, 64, 2, 2500),), (32, 64, 2, 2): ((250, 128, 2, 700),)}


def matrix(gen, rows, k, kp):
    """Codes with anything behind the k-th, and scales."""
    return torch.randint(-128, 128, (rows, kp), dtype=torch.int8, device="cuda", generator=gen), torch.rand(rows, device="cuda", generator=gen)


def columns(gen, n, k, kp):
    q = torch.randint(-127, 128, (n, kp), dtype=torch.int8, device="cuda", generator=gen)
    q[:, k:] = 0
    return q, torch.rand(n, device="cuda", generator=gen)


def value(q, s, w, ws):
    return (q.double() @ w.double().t()).float() * s[:, None] * ws[None, :]


@pytest.mark.parametrize("k", KS)
@pytest.mark.parametrize("form", ONE, ids=lambda f: "x".join(map(str, f)))
def test_one_matrix(gpu, form, k):
    m, rows = ONE[form]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m + rows + k)
    kp = bm.i8_row_bytes(k)
    (w, ws), (q, s) = matrix(gen, rows, k, kp), columns(gen, m, k, kp)
    dtype = (bm.F32, bm.F16, bm.BF16)[KS.index(k) % 3]
    y = torch.full((m, rows + 1), 7.0, dtype=TORCH[dtype], device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_i8_gemm(PTR(w), PTR(ws), rows, k, PTR(q), PTR(s), m, PTR(y), dtype, ld_y=rows + 1)
    gpu.sync()
    assert torch.equal(y[:, :rows], value(q, s, w, ws).to(TORCH[dtype]))
    assert (y[:, rows] == 7.0).all()
    clean(gpu)


@pytest.mark.parametrize("k", KS)
@pytest.mark.parametrize("own", (False, True), ids=("shared", "own"))
@pytest.mark.parametrize("form,size", [(f, s) for f, sizes in EXPERTS.items() for s in sizes], ids=lambda f: "x".join(map(str, f)))
def test_experts(gpu, form, size, own, k):
    m, n, top_k, rows = size
    rng = np.random.default_rng(m + n + rows + k)
    order, start, _ = tables(picks(rng, m, n, top_k, away=0.1), n)
    n_slots, listed = m * top_k, order.size
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m + n + rows + k)
    kp = bm.i8_row_bytes(k)
    (w, ws), (q, s) = matrix(gen, n * rows, k, kp), columns(gen, n_slots if own else m, k, kp)
    dtype = (bm.BF16, bm.F32, bm.F16)[KS.index(k) % 3]
    full = np.full(n_slots, 0x12345678, np.uint32)
    full[:listed] = order
    table, bounds = torch.from_numpy(full.view(np.int32)).cuda(), torch.from_numpy(start.view(np.int32)).cuda()
    col = torch.arange(listed, device="cuda") if own else torch.from_numpy(order.astype(np.int64)).cuda() // top_k
    y = torch.full((n_slots, rows), 7.0, dtype=TORCH[dtype], device="cuda")
    torch.cuda.synchronize()
    gpu.enqueue_i8_gemm_experts(PTR(w), PTR(ws), n, rows, k, PTR(q), PTR(s), None if own else PTR(table), PTR(bounds), n_slots, 0 if own else top_k, PTR(y), dtype)
    gpu.sync()
    for e in range(n):
        a, b = int(start[e]), int(start[e + 1])
        if b > a:
            of = slice(e * rows, (e + 1) * rows)
            assert torch.equal(y[a:b], value(q[col[a:b]], s[col[a:b]], w[of], ws[of]).to(TORCH[dtype])), f"expert {e}"
    assert (y[listed:] == 7.0).all()
    clean(gpu)


# (form, experts, rows): a table of 32767 slots
FAR = (((64, 64, 4, 2), 1, 40), ((256, 256, 8, 2), 1, 200), ((128, 128, 4, 2), 128, 100), ((64, 256, 4, 2), 300, 70), ((64, 128, 4, 2), 1000, 70))


def test_gathered_columns_far_into_the_tiles_reach(gpu):
    """Columns of 4.3 GB, the most that 32-bit offsets hold, behind an order, in every form of tiles that such a table takes."""
    k, cols = 131072, 32767
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    q, s = torch.randint(-127, 128, (cols, k), dtype=torch.int8, device="cuda", generator=gen), torch.rand(cols, device="cuda", generator=gen)
    listed = torch.tensor([cols - 1, 0, 16383, 16384, 16385, 20000, cols - 2] + list(range(cols - 60, cols - 20)), device="cuda")
    table = torch.full((cols,), 0x12345678, dtype=torch.int32, device="cuda")
    table[:listed.numel()] = listed.int()
    for form, n, rows in FAR:
        assert bm.i8_gemm_form(rows, k, cols, n, cols, 1) == form
        w, ws = torch.randint(-128, 128, (n * rows, k), dtype=torch.int8, device="cuda", generator=gen), torch.rand(n * rows, device="cuda", generator=gen)
        start = torch.full((n + 1,), 4, dtype=torch.int32, device="cuda")  # the first and the last expert's runs
        start[0], start[n] = 0, listed.numel()
        y = torch.full((cols, rows), 7.0, device="cuda")
        torch.cuda.synchronize()
        gpu.enqueue_i8_gemm_experts(PTR(w), PTR(ws), n, rows, k, PTR(q), PTR(s), PTR(table), PTR(start), cols, 1, PTR(y), bm.F32)
        gpu.sync()
        for e in {0, n - 1}:
            at = torch.arange(int(start[e]), int(start[e + 1]), device="cuda")
            of = slice(e * rows, (e + 1) * rows)
            assert torch.equal(y[at], value(q[listed[at]], s[listed[at]], w[of], ws[of])), form
        assert (y[listed.numel():] == 7.0).all()
        del w
    clean(gpu)
    torch.cuda.empty_cache()
