"""GPU tests of the experts' step in microscaled 4-bit floating point where its launches divide the work: experts with more tokens than one workgroup
takes, lines of down that several workgroups share, rows long enough for either form, the largest tables, weights that are not finite. The reference is formed in f64 on
the device from the same codes."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
import mx4_common as mx
from rows_common import HALF_STEP, NAMES, TORCH
from test_gpu_mx4 import KEPT, clean, gpu, picks  # noqa: F401 (a fixture)
from test_gpu_mx4_forms import rows_of, values_of

pytestmark = pytest.mark.gpu
PTR = torch.Tensor.data_ptr
DTYPES = pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)
SHAPES = {"gate": lambda h, f: (f, h), "up": lambda h, f: (f, h), "down": lambda h, f: (h, f)}


class Stack:
    def __init__(self, seed, n, hidden, ff):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.n, self.hidden, self.ff = n, hidden, ff
        self.dev = {}
        for name, of in SHAPES.items():
            rows, k = of(hidden, ff)
            w, s = rows_of(self.gen, n * rows, k, False)
            s -= torch.where(s == 255, 0, 4).to(torch.uint8)  # weights near 2^-8
            self.dev[name] = w, s

    def values(self, name, e):
        rows, k = SHAPES[name](self.hidden, self.ff)
        of = slice(e * rows, (e + 1) * rows)
        return values_of(self.dev[name][0][of], self.dev[name][1][of], k)

    def pointers(self):
        return [tuple(PTR(t) for t in self.dev[name]) for name in SHAPES]

    def rows(self, m, dtype, k=None):
        return torch.randn(m, k or self.hidden, device="cuda", generator=self.gen).to(TORCH[dtype])


def some_weights(gen, m, top_k):
    return torch.rand(m, top_k, device="cuda", generator=gen)


def step(g, stack, x, dtype, sel, wts, resid, y=None, work=None, rule=None):
    m, top_k = wts.shape
    if work is None:
        size = bm.mx4_moe_work(m, top_k, stack.hidden, stack.ff)
        work = torch.full((size + 4096,), 255, dtype=torch.uint8, device="cuda")
    if y is None:
        y = torch.full((m, stack.hidden), 7.0, dtype=TORCH[dtype], device="cuda")
    g.enqueue_mx4_moe(*stack.pointers(), stack.n, stack.hidden, stack.ff, PTR(x), dtype, m, PTR(sel), PTR(wts), top_k, None if resid is None else PTR(resid), PTR(y),
                      PTR(work), ld_x=x.stride(0), ld_resid=None if resid is None else resid.stride(0), ld_y=y.stride(0), rule=rule)
    return y, work


def ids(sel):
    """Picks on the device as the 32-bit words they are."""
    return torch.from_numpy(np.ascontiguousarray(sel).view(np.int32)).cuda()


def reference(stack, x, sel, wts, resid, kept):
    """mx4_common.moe, an expert at a time."""
    def steps(n):
        return (3 * -(-n // 32) + 64) * mx.STEP

    m, top_k = wts.shape
    xd, y = x.double(), torch.zeros(m, stack.hidden, dtype=torch.float64, device="cuda") if resid is None else resid.double()
    off, size = torch.zeros_like(y), y.abs()
    table = sel.cpu().numpy().view(np.uint32)
    for e in range(stack.n):
        t, s = np.nonzero(table == e)
        if t.size == 0:
            continue
        t, w = torch.from_numpy(t).cuda(), wts.double()[torch.from_numpy(t), torch.from_numpy(s)][:, None]
        xe, sums = xd[t], {}
        for name in ("gate", "up"):
            wv = stack.values(name, e).t().contiguous()
            sums[name] = xe @ wv, steps(stack.hidden) * (xe.abs() @ wv.abs())
        (g, dg), (u, du) = sums["gate"], sums["up"]
        silu = g / (1 + torch.exp(-g))
        h = silu * u
        dh = 1.1 * dg * (u.abs() + du) + (silu.abs() + 1.1 * dg) * du + kept * h.abs()  # silu's slope is below 1.1
        wv = stack.values("down", e).t().contiguous()
        d = h @ wv
        y = y.index_add(0, t, w * d)
        off = off.index_add(0, t, w.abs() * (dh @ wv.abs() + steps(stack.ff) * ((h.abs() + dh) @ wv.abs())))
        size = size.index_add(0, t, (w * d).abs())
    return y, off + (top_k + 1) * mx.STEP * (size + off)


def assert_step(y, dtype, stack, x, sel, wts, resid):
    exact, bound = reference(stack, x, sel, wts, resid, KEPT[dtype])
    off = HALF_STEP[dtype] * (exact.abs() + bound) + bound + (2.0 ** -25 if dtype == bm.F16 else 0.0)
    assert ((y.double() - exact).abs() <= off).all()


# (tokens, experts, top_k, hidden, ff). With top_k and hidden the number of workgroups that share down's lines goes from 1 to 8, by its lines and waves; hidden
# decides the forms at 2048 and 4096; few experts have many tokens each, more than one workgroup takes of them (2 to 8) and more than a tile of 16; stacks past 4 GiB.
SIZES = ((1, 128, 8, 2048, 768), (16, 128, 8, 2048, 768), (4, 64, 8, 1023, 1500), (16, 8, 1, 2048, 4096), (12, 40, 3, 2049, 2300), (5, 20, 8, 2600, 2048), (16, 64, 8, 4096, 1536),
         (16, 2, 2, 4096, 500), (2, 32, 4, 7168, 2048), (16, 24, 8, 8200, 300), (1, 300, 64, 512, 700), (16, 1024, 64, 64, 96), (64, 128, 8, 2048, 768), (64, 4, 4, 2048, 768),
         (64, 4, 2, 2100, 1100), (64, 1, 1, 2048, 4096), (64, 1, 1, 33, 20000), (40, 16, 8, 4500, 1100), (64, 2, 2, 4100, 1000), (64, 1024, 64, 96, 40), (64, 64, 64, 2080, 64),
         (17, 1000, 64, 40, 33), (33, 8, 8, 256, 16384), (2, 700, 8, 7168, 2048), (17, 2, 2, 33000, 300), (3, 2, 2, 300, 33000),
         (64, 4, 2, 4096, 300), (64, 2, 2, 2336, 100), (30, 8, 2, 3328, 40), (7, 5, 3, 2560, 33))


@DTYPES
@pytest.mark.parametrize("m,n,top_k,hidden,ff", SIZES)
def test_the_step_where_its_work_is_divided(gpu, dtype, m, n, top_k, hidden, ff):
    stack = Stack(m + n + hidden + ff, n, hidden, ff)
    rng = np.random.default_rng(m + n + top_k)
    x, resid = stack.rows(m, dtype), stack.rows(m, dtype)
    table = picks(rng, m, n, top_k, 0.05)
    sel, wts = ids(table), some_weights(stack.gen, m, top_k)
    torch.cuda.synchronize()
    y, work = step(gpu, stack, x, dtype, sel, wts, resid)
    gpu.sync()
    assert_step(y, dtype, stack, x, sel, wts, resid)
    assert (work[-4096:] == 255).all()
    again, _ = step(gpu, stack, x, dtype, sel, wts, resid, work=work)
    gpu.sync()
    assert torch.equal(y, again)
    held = resid.clone()
    torch.cuda.synchronize()
    step(gpu, stack, x, dtype, sel, wts, held, y=held)
    gpu.sync()
    assert torch.equal(y, held)
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("apart,shift", ((0, 0), (8, 0), (8, 8), (1, 0), (8, 1), (4, 2)))
@pytest.mark.parametrize("hidden", (1024, 2080, 4096))
def test_rows_on_every_kind_of_address(gpu, dtype, hidden, apart, shift):
    m, n, top_k, ff = 20, 9, 3, 100
    stack = Stack(3, n, hidden, ff)
    held = torch.full((m * (hidden + apart) + shift,), float("nan"), dtype=TORCH[dtype], device="cuda")
    x = held[shift:].view(m, hidden + apart)[:, :hidden]
    x.copy_(stack.rows(m, dtype))
    sel, wts = ids(picks(np.random.default_rng(4), m, n, top_k)), some_weights(stack.gen, m, top_k)
    torch.cuda.synchronize()
    y, _ = step(gpu, stack, x, dtype, sel, wts, None)
    gpu.sync()
    assert_step(y, dtype, stack, x, sel, wts, None)
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("m,n,top_k,hidden,ff", ((3, 4, 4, 2048, 768), (33, 3, 5, 2048, 512), (64, 2, 64, 2080, 96)))
def test_picks_of_the_same_expert_again_and_again(gpu, dtype, m, n, top_k, hidden, ff):
    """Tokens that pick an expert at several slots leave shares of it without tokens."""
    stack = Stack(77, n, hidden, ff)
    rng = np.random.default_rng(m)
    table = rng.integers(0, n, (m, top_k)).astype(np.uint32)
    table[::3] = 1
    x = stack.rows(m, dtype)
    sel, wts = ids(table), some_weights(stack.gen, m, top_k)
    torch.cuda.synchronize()
    y, _ = step(gpu, stack, x, dtype, sel, wts, None)
    gpu.sync()
    assert_step(y, dtype, stack, x, sel, wts, None)
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("m,hidden,ff", ((4, 2048, 768), (16, 4200, 300), (40, 300, 520), (64, 2200, 96)))
def test_no_picks_at_all(gpu, dtype, m, hidden, ff):
    stack = Stack(5, 3, hidden, ff)
    x, resid = stack.rows(m, dtype), stack.rows(m, dtype)
    sel, wts = ids(np.full((m, 2), bm.HOST_SLOT, np.uint32)), torch.full((m, 2), float("nan"), device="cuda")
    torch.cuda.synchronize()
    y, _ = step(gpu, stack, x, dtype, sel, wts, resid)
    z, _ = step(gpu, stack, x, dtype, sel, wts, None)
    gpu.sync()
    assert torch.equal(y, resid) and (z == 0).all()
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("byte", (255, 254))
@pytest.mark.parametrize("m,n,top_k,hidden,ff", ((2, 4, 2, 2048, 768), (16, 24, 4, 4100, 300), (40, 24, 4, 2048, 300), (64, 24, 4, 2300, 520)))
def test_weights_that_are_not_finite_stay_with_their_experts_tokens(gpu, dtype, name, byte, m, n, top_k, hidden, ff):
    """A block of an expert under the NaN scale, or with values past f32's range: every other token's sums are what they are without it."""
    stack = Stack(21, n, hidden, ff)
    rng = np.random.default_rng(9)
    table = picks(rng, m, n, top_k)
    if m == 2:
        table[:] = [[0, 1], [1, 2]]
    x, sel, wts = stack.rows(m, dtype), ids(table), some_weights(stack.gen, m, top_k)
    torch.cuda.synchronize()
    before, _ = step(gpu, stack, x, dtype, sel, wts, None)
    w, s = stack.dev[name]
    rows = SHAPES[name](hidden, ff)[0]
    e, row, block = 2, 19, 3
    w[e * rows + row, 16 * block:16 * (block + 1)] = 0x77  # all 6
    s[e * rows + row, block] = byte
    torch.cuda.synchronize()
    after, _ = step(gpu, stack, x, dtype, sel, wts, None)
    gpu.sync()
    users = torch.from_numpy((table == e).any(axis=1)).cuda()
    assert users.any() and not users.all()
    assert torch.equal(before[~users], after[~users])
    if name == "down":
        assert not torch.isfinite(after[users][:, row]).any()
        rest = torch.arange(hidden, device="cuda") != row
        assert torch.equal(before[users][:, rest], after[users][:, rest])
    else:
        assert not torch.isfinite(after[users]).any()
    clean(gpu)


@pytest.mark.parametrize("m,hidden,ff", ((2, 512, 256), (5, 2300, 96)))
def test_small_weights_under_large_values(gpu, m, hidden, ff):
    """Weights below f32's smallest ordinary number count in full."""
    stack = Stack(4, 2, hidden, ff)
    for name in ("gate", "up", "down"):
        s = stack.dev[name][1]
        s[s != 255] = 0
    x = stack.rows(m, bm.F32) * 2.0 ** 124
    sel, wts = ids(np.tile(np.array([[0, 1]], np.uint32), (m, 1))), torch.full((m, 2), 2.0 ** 126, device="cuda")
    torch.cuda.synchronize()
    y, _ = step(gpu, stack, x, bm.F32, sel, wts, None)
    gpu.sync()
    assert (y != 0).any()
    assert_step(y, bm.F32, stack, x, sel, wts, None)
    clean(gpu)


@DTYPES
def test_replays_and_a_second_context_give_the_same_bits(gpu, dtype):
    """Captured, replayed over other rows and picks between eager work, beside a second context with its own scratch on its own stream."""
    m, n, top_k, hidden, ff = 16, 32, 4, 2048, 768
    stack = Stack(8, n, hidden, ff)
    rng = np.random.default_rng(8)
    x, sel, wts = stack.rows(m, dtype), ids(picks(rng, m, n, top_k)), some_weights(stack.gen, m, top_k)
    other = bm.Gpu(0)
    torch.cuda.synchronize()
    _, w0 = step(gpu, stack, x, dtype, sel, wts, x)
    y, w1 = step(gpu, stack, x, dtype, sel, wts, x)
    z, w2 = step(other, stack, x, dtype, sel, wts, x)
    gpu.sync()
    other.sync()
    gpu.capture_begin()
    step(gpu, stack, x, dtype, sel, wts, x, y=y, work=w1)
    graph = gpu.capture_end()
    try:
        for turn in range(4):
            x.copy_(stack.rows(m, dtype))
            sel.copy_(ids(picks(rng, m, n, top_k, 0.2 * turn)))
            y.fill_(7.0)
            z.fill_(7.0)
            torch.cuda.synchronize()
            gpu.graph_launch(graph)
            for _ in range(3):
                step(other, stack, x, dtype, sel, wts, x, y=z, work=w2)
            gpu.sync()
            other.sync()
            eager, _ = step(gpu, stack, x, dtype, sel, wts, x, work=w0)
            gpu.sync()
            assert torch.equal(y, eager) and torch.equal(z, eager), turn
            assert_step(eager, dtype, stack, x, sel, wts, x)
    finally:
        gpu.graph_destroy(graph)
        other.close()
    clean(gpu)
