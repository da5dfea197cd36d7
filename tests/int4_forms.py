"""Products over 4-bit weights, one for each form of a launch."""

import ctypes

# (8-bit rows, gated, (few rows' kernel, 16-row tiles, 16-column tiles), contraction in parts, rows, columns, steps)
FORMS = [
    (False, False, (1, 1, 1), False, 5, 77, 3), (False, False, (1, 1, 2), False, 5, 4110, 2),
    (False, False, (1, 1, 4), False, 13, 8201, 2), (False, False, (1, 2, 4), False, 29, 20000, 2),
    (False, False, (0, 2, 8), False, 4100, 77, 2), (False, False, (0, 2, 8), True, 4100, 78, 10),
    (False, False, (0, 4, 8), False, 130, 20000, 2), (False, False, (0, 4, 8), True, 6200, 77, 10),
    (False, False, (0, 4, 16), False, 300, 20001, 2), (False, False, (0, 4, 16), True, 100, 20000, 27),
    (False, False, (0, 8, 16), False, 700, 12002, 2), (False, False, (0, 8, 16), True, 236, 8200, 56),
    (False, True, (1, 1, 2), False, 5, 21, 3), (False, True, (1, 1, 4), False, 13, 4110, 2),
    (False, True, (1, 2, 4), False, 29, 9000, 2), (False, True, (0, 2, 8), False, 45, 4110, 2),
    (False, True, (0, 2, 8), True, 45, 4111, 10), (False, True, (0, 4, 8), False, 300, 5000, 2),
    (False, True, (0, 4, 8), True, 45, 4110, 27), (False, True, (0, 4, 16), False, 130, 20000, 2),
    (False, True, (0, 4, 16), True, 4100, 77, 27), (False, True, (0, 8, 16), False, 200, 20000, 2),
    (False, True, (0, 8, 16), True, 236, 4110, 56),
    (True, False, (1, 1, 1), False, 5, 77, 3), (True, False, (1, 1, 2), False, 5, 4110, 2),
    (True, False, (1, 1, 4), False, 13, 8201, 2), (True, False, (1, 2, 4), False, 29, 20000, 2),
    (True, False, (0, 2, 8), False, 4100, 77, 2), (True, False, (0, 2, 8), True, 4100, 78, 10),
    (True, False, (0, 4, 8), False, 130, 20000, 2), (True, False, (0, 4, 8), True, 4100, 77, 27),
    (True, False, (0, 4, 16), False, 300, 20001, 2), (True, False, (0, 4, 16), True, 100, 8200, 27),
    (True, False, (0, 8, 16), False, 700, 12002, 2), (True, False, (0, 8, 16), True, 1367, 1040, 45),
    (True, True, (1, 1, 2), False, 5, 21, 3), (True, True, (1, 1, 4), False, 13, 4110, 2),
    (True, True, (1, 2, 4), False, 29, 9000, 2), (True, True, (0, 2, 8), False, 45, 4110, 2),
    (True, True, (0, 2, 8), True, 45, 4111, 10), (True, True, (0, 4, 8), False, 300, 5000, 2),
    (True, True, (0, 4, 8), True, 45, 4110, 27), (True, True, (0, 4, 16), False, 130, 20000, 2),
    (True, True, (0, 4, 16), True, 4100, 77, 27), (True, True, (0, 8, 16), False, 200, 20000, 2),
    (True, True, (0, 8, 16), True, 91, 8200, 45),
]


def cols_of(steps, group):
    """A contraction of `steps` steps of 128 whose last one has one group."""
    return 128 * (steps - 1) + group


def plan(eight, gated, rows, outs, cols, group, dtype):
    """((few, 16-row tiles, 16-column tiles), parts) of a launch."""
    from inferkernellab_amd import _lib

    a = _lib.Int4LinearArgs()
    a.rows, a.cols, a.out_cols, a.group, a.gated, a.dtype = rows, cols, outs, group, gated, dtype
    a.x_scales = 1 << 20 if eight else None
    v = _lib.load().ikl_int4_linear_plan(ctypes.byref(a))
    return (v >> 24, v >> 16 & 255, v >> 8 & 255), v & 255
