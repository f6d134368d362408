"""What the entry points of microscaled 4-bit floating point refuse, without a device: they look at their numbers before their context, so a call
with every number in order and no context comes as far as the context. Addresses below are never read. And the restatement that the
GPU tests compare with, against the form's definition value by value."""
import ctypes

import numpy as np
import pytest

import bloomery_amd as bm
import mx4_common as mx

P = 0x10000  # 16-byte aligned
LIB = bm.load_library()

# entry -> the arguments of a call in order but for its context
GOOD = {
    "bm_mx4_quantize": dict(x=P, type=bm.F16, ld_x=100, m=3, k=100, live=None, codes=P, scales=P),
    "bm_mx4_swiglu_quantize": dict(g=P, u=P, type=bm.F32, ld=101, m=3, k=100, rule=None, live=P, codes=P, scales=P),
    "bm_mx4_dequantize": dict(codes=P, scales=P, m=3, k=100, y=P, type=bm.BF16, ld_y=100),
    "bm_mx4_gemm": dict(w=P, w_scales=P, rows=7, k=100, codes=P, scales=P, m=3, y=P, y_type=bm.F32, ld_y=7),
    "bm_mx4_gemm_x": dict(w=P, w_scales=P, rows=7, k=100, x=P, x_type=bm.F32, ld_x=100, m=3, codes=P, scales=P, y=P, y_type=bm.BF16, ld_y=9),
    "bm_mx4_gemm_experts": dict(w=P, w_scales=P, n_experts=4, rows=7, k=100, codes=P, scales=P, n_cols=6, order=P, start=P, n_slots=12, top_k=2,
                                y=P, y_type=bm.F16, ld_y=7),
    "bm_mx4_moe": dict(wg=P, wg_scales=P, wu=P, wu_scales=P, wd=P, wd_scales=P, n_experts=4, hidden=100, ff=60, x=P, type=bm.BF16, ld_x=100,
                       n_tokens=3, sel=P, w=P, top_k=2, resid=2 * P, ld_resid=101, rule=None, y=P, ld_y=100, work=P),
}
WIDE = ("codes", "w", "w_scales", "wg", "wu", "wd", "wg_scales", "wu_scales", "wd_scales", "work")  # 16-byte aligned


def call(name, **changed):
    args = dict(GOOD[name], **changed)
    rc = getattr(LIB, name)(None, *args.values())
    return rc, LIB.bm_last_error(None).decode()


@pytest.mark.parametrize("name", GOOD)
def test_a_call_in_order_comes_as_far_as_its_context(name):
    rc, text = call(name)
    assert rc == bm.EARG and text == f"{name}: ctx is NULL"


@pytest.mark.parametrize("name", GOOD)
def test_pointers_that_are_missing_or_not_aligned(name):
    optional = {"bm_mx4_swiglu_quantize": ("live",), "bm_mx4_moe": ("resid",)}.get(name, ())
    for arg, value in GOOD[name].items():
        if value not in (P, 2 * P):
            continue
        rc, text = call(name, **{arg: None})
        if arg in optional:
            assert rc == bm.EARG and text.endswith("ctx is NULL"), arg
        else:
            assert rc == bm.EARG and "_dev is NULL" in text and name in text, (arg, text)
        rc, text = call(name, **{arg: value + 1})
        assert rc == bm.ESHAPE and "align" in text and name in text, (arg, text)
        if arg in WIDE and not (name == "bm_mx4_moe" and arg == "w") or arg == "scales":
            assert call(name, **{arg: value + 8})[0] == bm.ESHAPE, arg


@pytest.mark.parametrize("name", GOOD)
def test_types_and_lines(name):
    for arg in GOOD[name]:
        if arg in ("type", "x_type", "y_type"):
            for t in (2, 12, -1, 31):
                rc, text = call(name, **{arg: t})
                assert rc == bm.ETYPE and "element type" in text
        if arg.startswith("ld"):
            for ld in (1, 0, -40, (1 << 40) + 1):
                rc, text = call(name, **{arg: ld})
                assert rc == bm.ESHAPE and "apart" in text, (arg, ld, text)


@pytest.mark.parametrize("name", [n for n in GOOD if n != "bm_mx4_moe"])
def test_sizes_of_the_products(name):
    for k in (0, -16, 131073):
        assert call(name, k=k)[0] == bm.ESHAPE
    for m in (0, -1, (1 << 22) + 1):
        if "m" in GOOD[name]:
            assert call(name, m=m)[0] == bm.ESHAPE
        if "rows" in GOOD[name]:
            assert call(name, rows=m)[0] == bm.ESHAPE


def test_rows_in_bytes():
    for k, codes, scales in ((1, 16, 16), (32, 16, 16), (33, 32, 16), (512, 256, 16), (513, 272, 32), (2048, 1024, 64), (131072, 65536, 4096)):
        assert (bm.mx4_row_bytes(k), bm.mx4_row_scales(k)) == (codes, scales) == (mx.row_bytes(k), mx.row_scales(k))
    for k in (0, -1, 131073):
        assert bm.mx4_row_bytes(k) == bm.ESHAPE and bm.mx4_row_scales(k) == bm.ESHAPE


def test_runs_and_columns_of_the_experts_product():
    name = "bm_mx4_gemm_experts"
    for changed in (dict(n_slots=0), dict(n_slots=(1 << 22) + 1), dict(n_cols=0), dict(top_k=-1), dict(top_k=0, n_cols=11), dict(n_experts=0),
                    dict(n_experts=1025)):
        assert call(name, **changed)[0] == bm.ESHAPE, changed
    assert call(name, top_k=0, n_cols=12, order=None)[1].endswith("ctx is NULL")  # a column a slot: no order is read


def test_tokens_slots_and_sizes_of_the_step():
    name = "bm_mx4_moe"
    for changed in (dict(n_tokens=0), dict(n_tokens=65), dict(top_k=0), dict(top_k=65), dict(n_experts=0), dict(n_experts=1025), dict(hidden=0),
                    dict(hidden=131073, ld_x=140000, ld_y=140000, ld_resid=140000), dict(ff=0), dict(ff=131073), dict(y=2 * P, ld_y=102)):
        assert call(name, **changed)[0] == bm.ESHAPE, changed
    assert call(name, y=2 * P, ld_y=101)[1].endswith("ctx is NULL")  # onto the residual in place
    for m, top_k, hidden, ff in ((1, 1, 1, 1), (1, 8, 2048, 768), (64, 8, 7168, 2048), (64, 64, 100, 33), (3, 2, 131072, 131072)):
        assert 0 < bm.mx4_moe_work(m, top_k, hidden, ff) <= m * top_k * (8 * ff + 8 * hidden + 1024) + 65536
    for args in ((0, 1, 1, 1), (65, 1, 1, 1), (1, 65, 1, 1), (1, 1, 0, 1), (1, 1, 1, 131073)):
        assert bm.mx4_moe_work(*args) == bm.ESHAPE


def test_gate_rules():
    for name in ("bm_mx4_swiglu_quantize", "bm_mx4_moe"):
        for rule, limit, code in ((5, 0.0, bm.ETYPE), (-1, 0.0, bm.ETYPE), (bm.ACT_SITU, 0.0, bm.ESHAPE), (bm.ACT_SWIGLU_OAI, -1.0, bm.ESHAPE),
                                  (bm.ACT_SWIGLU_CLAMP, float("nan"), bm.ESHAPE), (bm.ACT_SILU_MUL, float("nan"), bm.EARG)):
            act = bm.GateAct(rule, limit)
            assert call(name, rule=ctypes.addressof(act))[0] == code, rule


def test_the_restatement_takes_the_nearest_value_and_the_even_code_between():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 64)) * np.exp(rng.standard_normal((40, 1)) * 8)
    x[0, :32] = np.ldexp(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] * 4), 11)
    codes, scales = mx.encode(x)
    v = mx.decode(codes, scales, 64)
    for r in range(40):
        for c in range(64):
            s = np.ldexp(1.0, int(scales[r, c // 32]) - 127)
            most = np.abs(x[r, c // 32 * 32:c // 32 * 32 + 32]).max()
            assert 4 * s <= most < 8 * s
            away = np.abs(np.abs(x[r, c]) / s - mx.LEVELS)
            best = np.flatnonzero(away == away.min())
            assert abs(v[r, c]) / s == mx.LEVELS[best[0] if len(best) == 1 or best[0] % 2 == 0 else best[1]]
    assert list(codes[0, :8]) == [0, 2, 2, 4, 4, 6, 6, 7]
    words, padded = mx.pack(codes, scales, 64, 0xAA)
    back = mx.unpack(words, padded, 64)
    assert np.array_equal(back[0], codes) and np.array_equal(back[1], scales) and padded.shape == (40, 16) and (padded[:, 2:] == 0xAA).all()
