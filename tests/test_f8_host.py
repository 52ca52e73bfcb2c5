"""What the operators over 8-bit float weights and over rows sorted by expert refuse before anything reaches a device. The entry points take any
non-null context here: they return before they look at it."""
import ctypes as C

import pytest

INVALID = -1
CTX = C.c_void_p(16)   # never dereferenced by a refused call


def _rows(pkg, **changes):
    return pkg.F8Rows(**{**dict(codes=4096, scale=4096, stride=256, scale_stride=8), **changes})


def _weight(pkg, **changes):
    return pkg.F8Weight(**{**dict(codes=8192, scale=4096, stride=256), **changes})


def _quantize(pkg, out=None, **changes):
    fields = dict(x=4096, x_stride=256, source=None, out=_rows(pkg, **(out or {})), dtype=0, rows=8, width=250, x_rows=8)
    return pkg.F8Quantize(**{**fields, **changes})


def _product(pkg, x=None, w=None, up=None, **changes):
    fields = dict(x=_rows(pkg, **(x or {})), w=_weight(pkg, **(w or {})), up=_weight(pkg, **(up or {})), offsets=None, y=4096, y_stride=128, y_scale=4096,
                  y_scale_stride=8, rows=8, n=100, k=250, experts=0, dtype=0, act=0, alpha=1.0, limit=7.0)
    return pkg.F8Product(**{**fields, **changes})


def _sort(pkg, **changes):
    return pkg.ExpertSort(**{**dict(choice=64, offsets=64, source=64, place=64, tokens=3, top=2, experts=8), **changes})


def _sum(pkg, **changes):
    fields = dict(y=4096, y_stride=128, place=64, weight=64, add=4096, add_stride=128, out=8192, out_stride=128, tokens=3, top=2, width=100, y_rows=6, y_dtype=0, dtype=0)
    return pkg.ExpertSum(**{**fields, **changes})


BAD_ROWS = [dict(codes=0), dict(codes=4104), dict(scale=0), dict(scale=4098), dict(stride=248), dict(stride=260), dict(stride=-256), dict(stride=1 << 40), dict(scale_stride=7),
            dict(scale_stride=1 << 40)]


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_rows_of_codes_that_are_refused(pkg, lib, bad):
    assert lib.swlm_op_f8_quantize_dev(CTX, _quantize(pkg, out=bad), None) == INVALID
    assert lib.swlm_op_f8_product_dev(CTX, _product(pkg, x=bad), None) == INVALID
    assert b"f8" in lib.swlm_last_error()


@pytest.mark.parametrize("bad", [dict(x=0), dict(x=4104), dict(x_stride=249), dict(x_stride=252), dict(x_stride=-256), dict(source=2), dict(dtype=3), dict(dtype=-1),
                                 dict(rows=-1), dict(rows=9), dict(rows=(1 << 30) + 1), dict(x_rows=-1), dict(x_rows=7), dict(width=0), dict(width=-5), dict(width=257)], ids=str)
def test_quantizations_that_are_refused(pkg, lib, bad):
    assert lib.swlm_op_f8_quantize_dev(CTX, _quantize(pkg, **bad), None) == INVALID


@pytest.mark.parametrize("bad", [dict(codes=0), dict(codes=8200), dict(scale=0), dict(scale=4097), dict(stride=240), dict(stride=257), dict(stride=0)], ids=str)
def test_matrices_that_are_refused(pkg, lib, bad):
    assert lib.swlm_op_f8_product_dev(CTX, _product(pkg, w=bad), None) == INVALID
    assert lib.swlm_op_f8_product_dev(CTX, _product(pkg, up=bad, act=1), None) == INVALID


@pytest.mark.parametrize("bad", [dict(y=0), dict(y=4100), dict(y_stride=96), dict(y_stride=100), dict(y_stride=-128), dict(dtype=4), dict(dtype=-1), dict(act=4), dict(act=-1),
                                 dict(rows=-1), dict(n=0), dict(k=0), dict(k=-8), dict(n=(1 << 24) + 16, y_stride=1 << 25), dict(experts=-1), dict(experts=1025, offsets=64),
                                 dict(experts=2), dict(experts=2, offsets=66), dict(dtype=3, y_scale=0), dict(dtype=3, y_scale=4097), dict(dtype=3, y_scale_stride=7),
                                 dict(act=3, alpha=float("nan")), dict(act=3, alpha=float("inf")), dict(act=3, limit=-1.0), dict(act=3, limit=float("nan")),
                                 dict(experts=1024, offsets=64, n=1 << 21, y_stride=1 << 21), dict(experts=1024, offsets=64, rows=1 << 29, n=4096, y_stride=4096, x=dict(scale_stride=1 << 29))],
                         ids=str)
def test_products_that_are_refused(pkg, lib, bad):
    assert lib.swlm_op_f8_product_dev(CTX, _product(pkg, **bad), None) == INVALID


@pytest.mark.parametrize("bad", [dict(choice=0), dict(offsets=0), dict(source=0), dict(place=0), dict(choice=66), dict(offsets=65), dict(source=67), dict(place=62), dict(tokens=-1),
                                 dict(top=0), dict(top=-1), dict(experts=0), dict(experts=1025), dict(tokens=1 << 29, top=3)], ids=str)
def test_sorts_that_are_refused(pkg, lib, bad):
    assert lib.swlm_op_expert_sort_dev(CTX, _sort(pkg, **bad), None) == INVALID


@pytest.mark.parametrize("bad", [dict(y=0), dict(y=4104), dict(y_stride=96), dict(y_stride=100), dict(place=0), dict(place=66), dict(weight=0), dict(weight=65), dict(add=4100),
                                 dict(add_stride=96), dict(out=0), dict(out=8200), dict(out_stride=97), dict(tokens=-1), dict(top=0), dict(width=0), dict(y_rows=-1), dict(y_dtype=3),
                                 dict(dtype=3), dict(dtype=-1), dict(tokens=1 << 29, top=3)], ids=str)
def test_sums_that_are_refused(pkg, lib, bad):
    assert lib.swlm_op_expert_sum_dev(CTX, _sum(pkg, **bad), None) == INVALID


def test_null_arguments(pkg, lib):
    assert lib.swlm_op_f8_quantize_dev(None, _quantize(pkg), None) == INVALID
    assert lib.swlm_op_f8_quantize_dev(CTX, None, None) == INVALID
    assert lib.swlm_op_f8_product_dev(None, _product(pkg), None) == INVALID
    assert lib.swlm_op_f8_product_dev(CTX, None, None) == INVALID
    assert lib.swlm_op_expert_sort_dev(None, _sort(pkg), None) == INVALID
    assert lib.swlm_op_expert_sort_dev(CTX, None, None) == INVALID
    assert lib.swlm_op_expert_sum_dev(None, _sum(pkg), None) == INVALID
    assert lib.swlm_op_expert_sum_dev(CTX, None, None) == INVALID
    assert lib.swlm_op_f8_status(None) == INVALID and lib.swlm_write_f8_status(None, 1) == INVALID


def test_what_has_no_rows_is_not_looked_at(pkg, lib):
    nothing = dict(codes=0, scale=0)
    assert lib.swlm_op_f8_quantize_dev(CTX, _quantize(pkg, out=nothing, x=0, rows=0), None) == 0
    assert lib.swlm_op_f8_quantize_dev(CTX, _quantize(pkg, out=nothing, x=0, x_rows=0, source=64), None) == 0
    assert lib.swlm_op_f8_product_dev(CTX, _product(pkg, x=nothing, w=nothing, y=0, rows=0, experts=3), None) == 0
    assert lib.swlm_op_expert_sum_dev(CTX, _sum(pkg, y=0, place=0, weight=0, out=0, tokens=0), None) == 0


def test_forms(lib):
    """The forms cover all columns; sizes out of range are refused."""
    form = (C.c_int * 3)()
    for rows in (1, 16, 17, 100, 777, 8192):
        for n in (1, 128, 4096, 5000):
            for k in (1, 129, 4100):
                for experts in (0, 7):
                    for gated in (0, 1):
                        assert lib.swlm_op_f8_product_form(rows, n, k, experts, gated, form) == 0
                        wide, tile, ctas = form
                        assert 0 <= wide <= n and (wide == n) == (tile == 0) and (tile == 0) == (ctas == 0)
                        assert tile in ((0, 16, 64) if gated else (0, 16, 32, 64, 128)) and ctas in (0, 1, 2, 4, 8) and wide % 128 * (n - wide) == 0
                        assert experts == 0 or wide in (0, n)
    for bad in ((0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1, 1, 1, -1), (1, 1, 1, 1025), ((1 << 30) + 1, 1, 1, 0)):
        assert lib.swlm_op_f8_product_form(*bad[:3], bad[3], 0, form) == INVALID
    assert lib.swlm_op_f8_product_form(1, 1, 1, 0, 0, None) == INVALID
