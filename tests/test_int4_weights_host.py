"""4-bit weights on the CPU: a packed weight's memory is its own; the largest
products that have a plan; rounding weights of any finite size."""

import ctypes

import pytest
import torch

from inferkernellab_amd import Int4Weight, _lib, pack_int4_weight, quantize_int4_weight

ALIGNMENT = {"codes": 16, "scales": 16, "zeros": 4}  # bytes, of ikl_int4_linear


@pytest.mark.parametrize("group,cols", [(32, 128), (64, 128), (128, 128), (128, 256)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
def test_a_packed_weight_shares_no_memory_with_what_it_was_packed_from(group, cols, gated, offset):
    """A contraction of one step leaves the scales and zero points in the order
    that they were given in; a buffer's slice may start anywhere."""
    groups = cols // group
    codes = torch.randint(0, 16, (32, cols)).to(torch.uint8)
    scales = (torch.rand(offset + 32 * groups) + 0.5)[offset:].view(32, groups)
    zeros = torch.randint(0, 16, (offset + 32 * groups,), dtype=torch.uint8)[offset:].view(32, groups)
    w = pack_int4_weight(codes, scales, zeros, group_size=group, gated=gated)
    for name, of in ALIGNMENT.items():
        assert getattr(w, name).data_ptr() % of == 0, name
        assert getattr(w, name).is_contiguous()
    want = w.dequantize()
    for t in (codes, scales, zeros):
        t.zero_()
    assert torch.equal(w.dequantize(), want)


def _linear(rows, cols, outs, **kw):
    a = _lib.Int4LinearArgs()
    a.x = a.codes = a.scales = a.y = 1 << 20  # an aligned address that nothing reads
    a.rows, a.cols, a.out_cols, a.x_stride, a.y_stride = rows, cols, outs, cols, outs
    a.group, a.dtype = 128, _lib.IKL_BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("rows,cols,outs,gated", [
    (18725, 4096, 14336, 0), (32768, 4096, 14336, 1), (4096, 4096, 128256, 0), (131072, 14336, 28672, 0),
    (1 << 24, 128, 4096, 0), ((1 << 31) - 128, 128, 16, 0)])
def test_products_of_many_rows_and_columns_have_a_plan(rows, cols, outs, gated, eight):
    """Long prompts, wide layers, a head's columns: as long as blocks of some form
    fit in a grid of fewer than 2^32 threads."""
    a = _linear(rows, cols, outs, gated=gated, x_scales=(1 << 20) if eight else None)
    assert _lib.load().ikl_int4_linear_workspace_size(ctypes.byref(a)) >= 0, _lib.last_error()


@pytest.mark.parametrize("rows,outs", [((1 << 31) + 1, 16), (1 << 40, 16), (1 << 62, 4096), ((1 << 63) - 1, 1)])
def test_products_that_no_grid_holds_are_refused(rows, outs):
    lib = _lib.load()
    a = _linear(rows, 128, outs)
    assert lib.ikl_int4_linear_workspace_size(ctypes.byref(a)) == _lib.IKL_EINVAL
    assert lib.ikl_int4_linear(ctypes.byref(a), None) == _lib.IKL_EINVAL
    assert "too many rows" in _lib.last_error()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("symmetric", [False, True])
def test_weights_up_to_the_largest_values_are_rounded_to_finite_ones(dtype, symmetric):
    """A group's range may be past its type's largest value; its steps are not.
    Half a step of each weight and half of its zero point, the step rounded to
    the type, in 64 bits."""
    most = torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(4)
    w = ((torch.rand(6, 64, generator=gen, dtype=torch.float64) * 2 - 1) * most).to(dtype)
    w[1, 0], w[1, 1], w[2, 0] = most, -most, -most
    g = w.double().view(6, -1, 32)
    q = quantize_int4_weight(w, group_size=32, symmetric=symmetric)
    if symmetric:
        step = g.abs().amax(-1, keepdim=True) / 7
    else:
        step = (g.amax(-1, keepdim=True).clamp(min=0) - g.amin(-1, keepdim=True).clamp(max=0)) / 15
    bound = step * ((0.5 if symmetric else 1.0) + 15 * torch.finfo(dtype).eps / 2 + 2.0**-20)
    # what a code stands for may lie half a step past fp32's largest value: codes less zero points, and steps
    units = Int4Weight(q.codes, torch.ones_like(q.scales), q.zeros, 6, 64, 32, False, torch.float32)
    steps = q.scales[0, :2, :6].t().double()[..., None]
    assert bool(steps.isfinite().all())
    assert bool(((units.dequantize().double().view(6, 2, 32) * steps - g).abs() <= bound).all())
