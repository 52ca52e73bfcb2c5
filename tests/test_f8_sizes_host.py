"""How large products over 8-bit float weights may be. The entry points take any non-null context here: they return before they look at it."""
import ctypes as C

import pytest

INVALID = -1
CTX = C.c_void_p(16)   # never dereferenced by a refused call


def _refusal(pkg, lib, rows, n, k, experts):
    """What a product of this size is told where nothing but its offsets (its matrix, without experts) is missing."""
    call = pkg.F8Product(x=pkg.F8Rows(codes=4096, scale=4096, stride=1 << 24, scale_stride=1 << 30), w=pkg.F8Weight(scale=4096, stride=1 << 24), y=4096, y_stride=1 << 24,
                         rows=rows, n=n, k=k, experts=experts)
    assert lib.swlm_op_f8_product_dev(CTX, call, None) == INVALID
    return lib.swlm_last_error()


# the last five are more than any memory holds, at the limit or next to it
TAKEN = [(524288, 8192, 2048, 1024), (524288, 14336, 4096, 256), (1 << 20, 4096, 4096, 1024), (1 << 24, 16384, 16, 0), (1 << 30, 1920, 1, 0), ((1 << 29) - 16 * 1024, 4096, 250, 1024),
         ((1 << 30) - 16, 1920, 1, 1), (1 << 30, 128, 1, 1024)]
REFUSED = [(1 << 30, 2048, 1, 0), ((1 << 29) - 16 * 1023, 4096, 250, 1024), (1 << 30, 1 << 24, 1, 0), (1 << 29, 4096, 250, 1024)]


@pytest.mark.parametrize("rows,n,k,experts", TAKEN)
def test_sizes_that_are_taken(pkg, lib, rows, n, k, experts):
    """An expert has its own rows only, so products of many experts and many rows are not refused for what all of them with all rows would come to."""
    assert b"offsets" in _refusal(pkg, lib, rows, n, k, experts) if experts else b"matrix" in _refusal(pkg, lib, rows, n, k, experts)
    assert lib.swlm_op_f8_product_form(rows, n, k, experts, 0, (C.c_int * 3)()) == 0


@pytest.mark.parametrize("rows,n,k,experts", REFUSED)
def test_sizes_that_are_refused(pkg, lib, rows, n, k, experts):
    """The call and the question after its form agree on what is too large."""
    assert b"too many" in _refusal(pkg, lib, rows, n, k, experts)
    assert lib.swlm_op_f8_product_form(rows, n, k, experts, 0, (C.c_int * 3)()) == INVALID


def test_matrices_of_too_many_rows_have_no_form(lib):
    """2^30 rows of all experts' matrices are the most, for the call and for the question after its form."""
    form = (C.c_int * 3)()
    assert lib.swlm_op_f8_product_form(8, 1 << 20, 128, 1024, 0, form) == 0
    assert lib.swlm_op_f8_product_form(8, (1 << 20) + 1, 128, 1024, 0, form) == INVALID
