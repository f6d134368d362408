"""GPU tests of the experts' step in microscaled 4-bit floating point over rows of more than 2048 values that end with a block (bf16's go straight into LDS): weights that
are not finite, no picks, replays beside a second context. Last lines of one block, of two, and whole ones."""
import numpy as np
import pytest
import torch

import bloomery_amd as bm
import test_gpu_mx4_step as steps
from test_gpu_mx4 import clean, gpu, picks  # noqa: F401 (a fixture)
from test_gpu_mx4_step import DTYPES, SHAPES, Stack, assert_step, ids, some_weights, step

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("byte", (255, 254))
@pytest.mark.parametrize("m,n,top_k,hidden,ff", ((2, 4, 2, 2080, 300), (16, 24, 4, 2112, 128), (40, 24, 4, 4096, 300), (64, 24, 4, 2560, 100)))
def test_weights_that_are_not_finite_stay_with_their_experts_tokens(gpu, dtype, name, byte, m, n, top_k, hidden, ff):
    steps.test_weights_that_are_not_finite_stay_with_their_experts_tokens(gpu, dtype, name, byte, m, n, top_k, hidden, ff)


@DTYPES
@pytest.mark.parametrize("m,hidden,ff", ((1, 2080, 64), (16, 4096, 300), (40, 2336, 520), (64, 2112, 96)))
def test_no_picks_at_all(gpu, dtype, m, hidden, ff):
    steps.test_no_picks_at_all(gpu, dtype, m, hidden, ff)


@DTYPES
@pytest.mark.parametrize("m,n,top_k,hidden,ff", ((16, 32, 4, 2080, 200), (40, 6, 3, 4096, 100)))
def test_replays_beside_a_second_context(gpu, dtype, m, n, top_k, hidden, ff):
    """Captured, replayed over other rows and picks, beside a second context with its own scratch on its own stream."""
    stack = Stack(18, n, hidden, ff)
    rng = np.random.default_rng(18)
    x, sel, wts = stack.rows(m, dtype), ids(picks(rng, m, n, top_k)), some_weights(stack.gen, m, top_k)
    other = bm.Gpu(0)
    torch.cuda.synchronize()
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
            assert torch.equal(y, z), turn
            assert_step(y, dtype, stack, x, sel, wts, x)
    finally:
        gpu.graph_destroy(graph)
        other.close()
    clean(gpu)
