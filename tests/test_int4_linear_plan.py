"""The rule between the forms of a product over 4-bit weights. On the CPU."""

import ctypes

import pytest

from inferkernellab_amd import _lib
from tests.int4_forms import FORMS, cols_of, plan

KERNELS = {(1, 1, 1), (1, 1, 2), (1, 1, 4), (1, 2, 4), (0, 2, 8), (0, 4, 8), (0, 4, 16), (0, 8, 16)}


@pytest.mark.parametrize("eight,gated,form,parts,rows,outs,steps", FORMS)
def test_the_products_that_the_forms_are_tested_by_take_them(eight, gated, form, parts, rows, outs, steps):
    """A changed rule may not leave a form without its test."""
    for group in (32, 64, 128):
        for dtype in (_lib.IKL_BF16, _lib.IKL_F16, *((_lib.IKL_F32,) if eight else ())):
            taken, split = plan(eight, gated, rows, outs, cols_of(steps, group), group, dtype)
            assert (taken, split > 1) == (form, parts), (group, dtype, taken, split)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_every_form_has_its_products(eight, gated):
    """The few rows' kernel by one column tile has no pair of a gate's and an up
    projection's."""
    have = {(form, parts) for e, g, form, parts, *_ in FORMS if (e, g) == (eight, gated)}
    assert have == {(f, p) for f in KERNELS for p in (False, True)
                    if not (f[0] and p) and not (gated and f == (1, 1, 1))}


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_no_other_form_is_taken(eight, gated):
    for rows in (1, 2, 16, 17, 31, 32, 33, 64, 65, 100, 128, 200, 257, 513, 1000, 2047, 4096, 10000, 100000):
        for outs in (1, 16, 100, 512, 1024, 2048, 4096, 5001, 14336, 28672, 128256):
            for cols in (128, 256, 1024, 2048, 4096, 5632, 14336, 28672):
                form, parts = plan(eight, gated, rows, outs, cols, 128, _lib.IKL_BF16)
                assert form in KERNELS and 1 <= parts <= 16
                assert parts == 1 or (not form[0] and 2 * parts <= cols // 128)


def test_plans_refuse_and_no_rows_have_none():
    lib = _lib.load()
    a = _lib.Int4LinearArgs()
    a.rows, a.cols, a.out_cols, a.group, a.dtype = 4, 96, 16, 64, _lib.IKL_BF16
    assert lib.ikl_int4_linear_plan(ctypes.byref(a)) < 0 and lib.ikl_int4_linear_plan(None) < 0
    a.cols, a.rows = 64, 0
    assert lib.ikl_int4_linear_plan(ctypes.byref(a)) == 0
