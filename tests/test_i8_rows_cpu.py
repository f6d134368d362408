"""What the 8-bit products' and the sorted rows' entry points refuse, without a device: they look at their numbers before their
context, so a call with every number in order and no context comes as far as the context. Addresses below are never read."""
import ctypes

import pytest

import bloomery_amd as bm

P = 0x10000  # 16-byte aligned
LIB = bm.load_library()

# entry -> the arguments of a call in order but for its context
GOOD = {
    "bm_expert_sort": dict(sel=P, n_tokens=600, top_k=8, n_experts=16, x=P, type=bm.BF16, ld_x=40, width=33, order=P, start=P, place=P, rows=P,
                           ld_rows=33, work=P),
    "bm_expert_sort_grad": dict(d_rows=P, type=bm.F32, ld_rows=33, place=P, n_tokens=5, top_k=2, width=33, dx=P, ld_dx=34),
    "bm_expert_combine": dict(rows=P, type=bm.F16, ld_rows=8, place=P, w=P, resid=P, ld_resid=8, n_tokens=5, top_k=64, width=8, y=P, ld_y=8),
    "bm_expert_combine_grad": dict(dy=P, type=bm.BF16, ld_dy=8, rows=P, ld_rows=8, place=P, w=P, n_tokens=5, top_k=1, width=7, d_rows=P,
                                   ld_d_rows=7, d_w=P),
    "bm_i8_quantize": dict(x=P, type=bm.F16, ld_x=100, m=3, k=100, live=None, codes=P, scales=P),
    "bm_i8_swiglu_quantize": dict(g=P, u=P, type=bm.F32, ld=101, m=3, k=100, rule=None, live=P, codes=P, scales=P),
    "bm_i8_gemm": dict(w=P, w_scales=P, rows=7, k=100, codes=P, scales=P, m=3, y=P, y_type=bm.F32, ld_y=7),
    "bm_i8_gemm_x": dict(w=P, w_scales=P, rows=7, k=100, x=P, x_type=bm.F32, ld_x=100, m=3, codes=P, scales=P, y=P, y_type=bm.BF16, ld_y=9),
    "bm_i8_gemm_experts": dict(w=P, w_scales=P, n_experts=4, rows=7, k=100, codes=P, scales=P, n_cols=6, order=P, start=P, n_slots=12, top_k=2,
                               y=P, y_type=bm.F16, ld_y=7),
}
TYPES = {name: [k for k in args if k in ("type", "x_type", "y_type")] for name, args in GOOD.items()}


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
    optional = {"bm_i8_swiglu_quantize": ("live",), "bm_expert_combine": ("resid",)}.get(name, ())
    for arg, value in GOOD[name].items():
        if value != P:
            continue
        rc, text = call(name, **{arg: None})
        if arg in optional:
            assert rc == bm.EARG and text.endswith("ctx is NULL"), arg
        else:
            assert rc == bm.EARG and "_dev is NULL" in text and name in text, (arg, text)
        rc, text = call(name, **{arg: P + 1})
        assert rc == bm.ESHAPE and "align" in text and name in text, (arg, text)
        if arg in ("codes", "w") and name.startswith("bm_i8"):
            assert call(name, **{arg: P + 8})[0] == bm.ESHAPE, arg


@pytest.mark.parametrize("name", GOOD)
def test_types_and_lines(name):
    for arg in TYPES[name]:
        for t in (2, 12, -1, 31):
            rc, text = call(name, **{arg: t})
            assert rc == bm.ETYPE and "element type" in text
    for arg, value in GOOD[name].items():
        if arg.startswith("ld"):
            for ld in (1, 0, -40, (1 << 40) + 1):
                rc, text = call(name, **{arg: ld})
                assert rc == bm.ESHAPE and "apart" in text, (arg, ld, text)


@pytest.mark.parametrize("name", [n for n in GOOD if "expert_" in n])
def test_tokens_slots_and_experts(name):
    for changed in (dict(n_tokens=0), dict(n_tokens=-1), dict(top_k=0), dict(top_k=65), dict(n_tokens=(1 << 22) + 1, top_k=1),
                    dict(n_tokens=1 << 30, top_k=8)):
        if "n_tokens" in GOOD[name]:
            assert call(name, **changed)[0] == bm.ESHAPE, changed
    if "n_experts" in GOOD[name]:
        for n in (0, -3, 1025):
            assert call(name, n_experts=n)[0] == bm.ESHAPE
    if "width" in GOOD[name]:
        for w in (0, -1, (1 << 24) + 1):
            assert call(name, width=w)[0] == bm.ESHAPE


def test_sort_scratch_and_the_tables_alone():
    assert bm.expert_sort_work(4096, 1024) == 0 and bm.expert_sort_work(1, 1) == 0
    assert bm.expert_sort_work(0, 4) == bm.ESHAPE and bm.expert_sort_work(4, 1025) == bm.ESHAPE and bm.expert_sort_work((1 << 22) + 1, 4) == bm.ESHAPE
    for n in (4097, 5000, 65536, 100000, 1 << 22):
        for experts in (1, 7, 128, 1024):
            assert 0 < bm.expert_sort_work(n, experts) <= -(-n // 512) * experts
    none = dict(x=None, rows=None, type=99, width=-1, ld_x=-5, ld_rows=0)  # not looked at
    assert call("bm_expert_sort", **none)[1].endswith("ctx is NULL")
    assert call("bm_expert_sort", x=None)[0] == bm.EARG and call("bm_expert_sort", rows=None)[0] == bm.EARG  # one without the other
    assert call("bm_expert_sort", n_tokens=512, work=None)[1].endswith("ctx is NULL")  # 4096 slots need none


@pytest.mark.parametrize("name", [n for n in GOOD if n.startswith("bm_i8")])
def test_sizes_of_the_products(name):
    for k in (0, -16, 131073):
        assert call(name, k=k)[0] == bm.ESHAPE
    for m in (0, -1, (1 << 22) + 1):
        if "m" in GOOD[name]:
            assert call(name, m=m)[0] == bm.ESHAPE
        if "rows" in GOOD[name]:
            assert call(name, rows=m)[0] == bm.ESHAPE
    assert bm.i8_row_bytes(1) == 16 and bm.i8_row_bytes(16) == 16 and bm.i8_row_bytes(17) == 32 and bm.i8_row_bytes(131072) == 131072
    assert bm.i8_row_bytes(0) == bm.ESHAPE and bm.i8_row_bytes(131073) == bm.ESHAPE


def test_runs_and_columns_of_the_experts_product():
    name = "bm_i8_gemm_experts"
    for changed in (dict(n_slots=0), dict(n_slots=(1 << 22) + 1), dict(n_cols=0), dict(top_k=-1), dict(top_k=0, n_cols=11)):
        assert call(name, **changed)[0] == bm.ESHAPE, changed
    assert call(name, top_k=0, n_cols=12, order=None)[1].endswith("ctx is NULL")  # a column a slot: no order is read


def test_gate_rules():
    for rule, limit, code in ((5, 0.0, bm.ETYPE), (-1, 0.0, bm.ETYPE), (bm.ACT_SITU, 0.0, bm.ESHAPE), (bm.ACT_SWIGLU_OAI, -1.0, bm.ESHAPE),
                              (bm.ACT_SWIGLU_CLAMP, float("nan"), bm.ESHAPE), (bm.ACT_SILU_MUL, float("nan"), bm.EARG)):
        act = bm.GateAct(rule, limit)
        assert call("bm_i8_swiglu_quantize", rule=ctypes.addressof(act))[0] == code, rule
