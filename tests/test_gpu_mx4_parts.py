"""GPU tests of what the experts' step in microscaled 4-bit floating point keeps of its values: h in sixteen bits at least whatever the rows' type, infinities as
infinities. Weights are chosen so that every sum but the one looked at is exact; the references are formed in 64 bits on the host."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
import mx4_common as mx
from rows_common import HALF_STEP, NAMES, TORCH
from test_gpu_mx4 import clean, gpu  # noqa: F401 (a fixture)
from test_gpu_mx4_step import ids, step

pytestmark = pytest.mark.gpu
PTR = torch.Tensor.data_ptr
DTYPES = pytest.mark.parametrize("dtype", (bm.F32, bm.F16, bm.BF16), ids=NAMES.get)
ONE, MINUS_ONE = 2, 10  # codes


class Given:
    """Experts' matrices from codes: gate and up n x ff x hidden, down n x hidden x ff, a code 0 .. 15 each; every scale 1 (byte 127) until it is changed."""

    def __init__(self, gate, up, down):
        self.n, self.ff, self.hidden = gate.shape
        self.dev = {}
        for name, codes in (("gate", gate), ("up", up), ("down", down)):
            n, rows, k = codes.shape
            wide = np.zeros((n * rows, 2 * mx.row_bytes(k)), np.uint8)
            wide[:, :k] = codes.reshape(-1, k)
            w, s = mx.pack(wide, np.full((n * rows, -(-k // 32)), 127, np.uint8), k)
            self.dev[name] = torch.from_numpy(w).cuda(), torch.from_numpy(s).cuda()

    def pointers(self):
        return [tuple(PTR(t) for t in self.dev[name]) for name in ("gate", "up", "down")]


def rows(x, dtype):
    return torch.from_numpy(np.asarray(x, np.float32)).to(TORCH[dtype]).cuda()


def run(g, stack, x, dtype, sel):
    """The step of one slot a token, of weight 1."""
    y, _ = step(g, stack, x, dtype, ids(sel.astype(np.uint32)[:, None]), torch.ones(len(sel), 1, device="cuda"), None)
    g.sync()
    return y


# h's parts: the first two cut to 8 bits of mantissa, the last rounded to 8. Two parts: what the cut leaves is below 2^-7 of the value's power of two, its rounding off by
# at most 2^-9 of that. The rule's f32 operations: 2^-20.
KEPT = {bm.F32: 2.0 ** -20, bm.F16: 2.0 ** -16 + 2.0 ** -20, bm.BF16: 2.0 ** -16 + 2.0 ** -20}


# tokens, experts, hidden, ff: every form of up (rows up to 2048; longer ones by type and whether they end with a block) and of down (by hidden, tokens, and where several
# workgroups share its lines), experts with one token to 64
@DTYPES
@pytest.mark.parametrize("m,n,hidden,ff", ((1, 1, 64, 64), (5, 2, 512, 96), (16, 2, 2048, 64), (16, 3, 2056, 96), (40, 2, 2080, 64), (64, 1, 4096, 96), (64, 20, 300, 512),
                                           (20, 2, 7168, 64), (8, 8, 512, 4096), (64, 8, 256, 4096)))
def test_h_keeps_sixteen_bits(gpu, dtype, m, n, hidden, ff):
    """A row of gate and of up meets one value of a token, a row of down takes the difference of two h: it shows what each was held in."""
    rng = np.random.default_rng(m + hidden + ff)
    gate, up, down = np.zeros((n, ff, hidden), np.uint8), np.zeros((n, ff, hidden), np.uint8), np.zeros((n, hidden, ff), np.uint8)
    e, f, r = np.arange(n)[:, None], np.arange(ff)[None, :], np.arange(hidden)[None, :]
    gi, ui, gc, uc = rng.integers(0, hidden, (n, ff)), rng.integers(0, hidden, (n, ff)), rng.integers(1, 7, (n, ff)), rng.integers(1, 16, (n, ff))
    gate[e, f, gi], up[e, f, ui] = gc, uc
    plus = rng.integers(0, ff, (n, hidden))
    minus = (plus + rng.integers(1, ff, (n, hidden))) % ff
    down[e, r, plus], down[e, r, minus] = ONE, MINUS_ONE
    x = rng.integers(1, 33, (m, hidden)) / 8.0 * rng.choice([-1.0, 1.0], (m, hidden))  # six bits: whole in every type, and so are g and u
    sel = np.arange(m) % n
    y = run(gpu, Given(gate, up, down), rows(x, dtype), dtype, sel).double().cpu().numpy()
    value = np.concatenate([mx.LEVELS, -mx.LEVELS])
    t = np.arange(m)[:, None]
    h = mx.rule_value(value[gc[sel]] * x[t, gi[sel]], value[uc[sel]] * x[t, ui[sel]])
    a, b = h[t, plus[sel]], h[t, minus[sel]]
    bound = (KEPT[dtype] + 8 * mx.STEP) * (np.abs(a) + np.abs(b))  # eight f32 steps for the six parts' sum
    off = HALF_STEP[dtype] * (np.abs(a - b) + bound) + bound + (2.0 ** -25 if dtype == bm.F16 else 0.0)
    assert (np.abs(y - (a - b)) <= off).all()
    clean(gpu)


def signed(rng, hidden, ff):
    """Gate and up of ones, and down's rows of any sizes, a sign a row; and the signs."""
    sign = np.where(rng.random(hidden) < 0.5, -1.0, 1.0)
    down = (rng.integers(1, 8, (1, hidden, ff)) + np.where(sign < 0, 8, 0)[None, :, None]).astype(np.uint8)
    return np.full((1, ff, hidden), ONE, np.uint8), np.full((1, ff, hidden), ONE, np.uint8), down, sign


# up: short; long and ragged; long and whole (bf16: straight into LDS), its last line of 1, 2 and 8 blocks. down: 16 and 32 rows a workgroup, up to 16 tokens and more
SIZES = ((3, 64), (20, 300), (3, 2048), (20, 2056), (3, 2080), (20, 2112), (3, 2304), (40, 4096), (3, 4100))


@DTYPES
@pytest.mark.parametrize("m,hidden", SIZES)
def test_an_infinite_h_stays_infinite(gpu, dtype, m, hidden):
    """Finite sums whose product passes f32's range, of every second token."""
    rng, ff = np.random.default_rng(hidden), 72
    gate, up, down, sign = signed(rng, hidden, ff)
    gate[..., 1:], up[..., 1:] = 0, 0
    stack = Given(gate, up, down)
    for name in ("gate", "up"):
        stack.dev[name][1][:, 0] = 127 + 70
    x = np.zeros((m, hidden))
    x[::2, 0] = 1.0
    y = run(gpu, stack, rows(x, dtype), dtype, np.zeros(m)).double().cpu().numpy()
    assert (y[::2] == np.inf * sign).all() and (y[1::2] == 0).all()
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("m,hidden", SIZES)
def test_an_infinite_value_of_a_token(gpu, dtype, m, hidden):
    """At the row's ends and between them, alone and under either sign: the token's sums are infinite, the others' what they are without it."""
    rng, ff = np.random.default_rng(hidden), 40
    gate, up, down, sign = signed(rng, hidden, ff)
    for minus in (False, True):
        if minus:
            gate[:], up[:] = MINUS_ONE, MINUS_ONE
        stack = Given(gate, up, down)
        x = np.where(minus, -1.0, 1.0) * rng.integers(1, 9, (m, hidden)) / 2.0 ** 14
        before = run(gpu, stack, rows(x, dtype), dtype, np.zeros(m))
        assert torch.isfinite(before).all()
        for at in (0, 5, hidden // 2, hidden - 1):
            z = x.copy()
            z[1, at] *= np.inf
            after = run(gpu, stack, rows(z, dtype), dtype, np.zeros(m))
            assert (after[1].double().cpu().numpy() == np.inf * sign).all(), at
            rest = torch.arange(m) != 1
            assert torch.equal(before[rest], after[rest]), at
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("m,hidden", [s for s in SIZES if s[1] > 2048])
def test_an_infinite_value_where_the_last_line_begins(gpu, dtype, m, hidden):
    """Whatever a kernel reads in the place of what is behind a row's end, it counts for nothing."""
    rng, ff = np.random.default_rng(hidden), 40
    gate, up, down, sign = signed(rng, hidden, ff)
    stack = Given(gate, up, down)
    x = rng.integers(1, 9, (m, hidden)) / 2.0 ** 14
    for at in range(256 * ((hidden - 1) // 256), hidden, 7):
        z = x.copy()
        z[1, at] = np.inf
        y = run(gpu, stack, rows(z, dtype), dtype, np.zeros(m)).double().cpu().numpy()
        assert (y[1] == np.inf * sign).all() and np.isfinite(np.delete(y, 1, 0)).all(), at
    clean(gpu)


@DTYPES
@pytest.mark.parametrize("byte", (253, 254))
@pytest.mark.parametrize("name", ("gate", "up"))
@pytest.mark.parametrize("m,hidden", SIZES)
def test_a_code_past_f32s_range_is_an_infinity(gpu, dtype, name, byte, m, hidden):
    """Against values that a first part holds whole as well as others."""
    rng, ff = np.random.default_rng(hidden), 72
    gate, up, down, sign = signed(rng, hidden, ff)
    row = {"gate": gate, "up": up}[name][0, 3]
    row[32:64] = 0
    row[40] = 7
    x = rng.choice([1.0, 1.5, 1.0 + 2.0 ** -7, 1.0 + 2.0 ** -10, 1.0 + 2.0 ** -23], (m, hidden)) / 2.0 ** 13  # (f16: ordinary numbers)
    stack = Given(gate, up, down)
    assert torch.isfinite(run(gpu, stack, rows(x, dtype), dtype, np.zeros(m))).all()
    stack.dev[name][1][3, 1] = byte
    y = run(gpu, stack, rows(x, dtype), dtype, np.zeros(m)).double().cpu().numpy()
    assert (y == np.inf * sign).all()
    clean(gpu)


# experts with up to four tokens, up to eight (two groups side by side in a matrix instruction's columns), and more; several lines of down
@DTYPES
@pytest.mark.parametrize("byte", (253, 254))
@pytest.mark.parametrize("m,hidden,ff", ((3, 64, 72), (7, 64, 72), (8, 4096, 300), (16, 300, 600), (20, 2056, 72), (40, 4096, 600), (64, 512, 2048)))
def test_a_code_of_down_past_f32s_range_is_an_infinity(gpu, dtype, byte, m, hidden, ff):
    """Its row alone is infinite, for every token, by the code's sign."""
    rng = np.random.default_rng(hidden)
    gate, up, down, _ = signed(rng, hidden, ff)
    for row, code in ((5, 7), (6, 15)):
        down[0, row, 32:64] = 0
        down[0, row, 40] = code
    x = rng.choice([1.0, 1.5, 1.0 + 2.0 ** -7, 1.0 + 2.0 ** -10, 1.0 + 2.0 ** -23], (m, hidden)) / 2.0 ** 13  # (f16: ordinary numbers)
    stack = Given(gate, up, down)
    before = run(gpu, stack, rows(x, dtype), dtype, np.zeros(m))
    assert torch.isfinite(before).all()
    stack.dev["down"][1][5:7, 1] = byte
    after = run(gpu, stack, rows(x, dtype), dtype, np.zeros(m))
    assert (after[:, 5] == np.inf).all() and (after[:, 6] == -np.inf).all()
    rest = torch.ones(hidden, dtype=torch.bool, device="cuda")
    rest[5:7] = False
    assert torch.equal(before[:, rest], after[:, rest])
    clean(gpu)
