"""Which form the products in microscaled 4-bit floating point take, without a device: the sizes that the GPU tests run lead to the forms that they mean to hold, and
together to every form that there is."""
import pytest

import bloomery_amd as bm
from test_gpu_mx4_forms import EXPERTS, KS, ONE

FORMS = {(16, 16, 8, 4), (16, 32, 3, 4), (32, 32, 4, 4), (32, 64, 2, 2), (64, 64, 4, 2), (128, 128, 4, 2), (256, 128, 8, 2), (256, 256, 8, 2)}


@pytest.mark.parametrize("k", KS)
def test_the_gpu_tests_sizes_take_their_forms(k):
    for form, sizes in ONE.items():
        for m, rows in sizes:
            assert bm.mx4_gemm_form(rows, k, m) == form, (m, rows)
    for form, sizes in EXPERTS.items():
        for m, n, top_k, rows in sizes:
            assert bm.mx4_gemm_form(rows, k, m, n, m * top_k, top_k) == form, (m, n, top_k, rows)
            assert bm.mx4_gemm_form(rows, k, m * top_k, n, m * top_k, 0) == form
    assert set(ONE) | set(EXPERTS) == FORMS


def test_the_lines_of_the_gpu_tests_sizes():
    """One line alone, two, and odd and even numbers of them; last lines of one block and of all eight."""
    lines = [-(-k // 256) for k in KS]
    assert lines == [1, 1, 2, 3, 4, 6, 9, 10, 13]
    assert {-(-k // 32) - 8 * (n - 1) for k, n in zip(KS, lines)} >= {1, 2, 8}


def test_every_size_has_one_of_these_forms():
    seen = set()
    octaves = [1 << b for b in range(0, 23, 2)] + [(1 << b) - 1 for b in range(4, 23, 3)]
    for rows in octaves:
        for m in octaves:
            for k in (16, 1000, 2048, 131072):
                seen.add(bm.mx4_gemm_form(rows, k, m))
                for n in (1, 7, 64, 1000):
                    seen.add(bm.mx4_gemm_form(rows, k, m, n, m, 0))
                    seen.add(bm.mx4_gemm_form(rows, k, max(1, m // 2), n, m, 2))
    assert seen <= FORMS


def test_gathered_columns_past_32_bits_take_the_form_with_whole_addresses():
    at = (1 << 32) // 2048
    assert bm.mx4_gemm_form(700, 4096, at - 1, 8, 4000, 2) == bm.mx4_gemm_form(700, 4096, 4000, 8, 4000, 2)
    assert bm.mx4_gemm_form(700, 4096, at, 8, 4000, 2) == (16, 32, 3, 4)
    assert bm.mx4_gemm_form(700, 4096, at, 8, 4000, 0) == bm.mx4_gemm_form(700, 4096, 4000, 8, 4000, 0)


def test_sizes_that_the_entries_refuse():
    lib = bm.load_library()
    for args in ((0, 0, 64, 5, 0, 0), (0, 64, 0, 5, 0, 0), (0, 64, 131073, 5, 0, 0), (0, 64, 64, 0, 0, 0), (0, 64, 64, (1 << 22) + 1, 0, 0), (-1, 64, 64, 5, 5, 0),
                 (1025, 64, 64, 5, 5, 0), (4, 64, 64, 5, 0, 1), (4, 64, 64, 5, 6, 0), (4, 64, 64, 5, 6, -1), (4, 64, 64, 5, (1 << 22) + 1, 2)):
        assert lib.bm_mx4_gemm_form(*args) == bm.ESHAPE, args
