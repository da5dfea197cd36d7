"""What the quantised operators refuse, before anything is launched (pointers
are addresses that nothing reads), and the layout of 4-bit weights, which needs
no GPU."""

import ctypes

import pytest
import torch

from inferkernellab_amd import Int4Weight, Int8Rows, _lib, pack_int4_weight, quantize_int4_weight

P = 1 << 20  # an aligned address


def _set(a, given):
    for k, v in given.items():
        setattr(a, k, v)
    return a


def _rows(**kw):
    a = _lib.Int8RowsArgs()
    a.x = a.codes = a.scales = P
    a.rows, a.cols, a.x_stride, a.group, a.dtype = 4, 256, 256, 64, _lib.IKL_BF16
    return _set(a, kw)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=0), dict(cols=96), dict(group=16), dict(group=0), dict(dtype=3),
                                 dict(x=0), dict(codes=0), dict(scales=0), dict(x=P + 8), dict(codes=P + 8),
                                 dict(scales=P + 2), dict(up=P + 2), dict(x_stride=257), dict(up=P, up_stride=4),
                                 dict(rows=1 << 31), dict(rows=1 << 62)], ids=str)
def test_rows_refuse(bad):
    lib = _lib.load()
    assert lib.ikl_quantize_rows_int8(ctypes.byref(_rows(**bad)), None) in (_lib.IKL_EINVAL, _lib.IKL_EUNSUPPORTED)
    assert "int8 rows" in _lib.last_error()


def _norm(**kw):
    a = _lib.NormInt8Args()
    a.x = a.weight = a.codes = a.scales = P
    a.rows, a.cols, a.x_stride, a.group, a.dtype, a.eps = 4, 256, 256, 64, _lib.IKL_BF16, 1e-6
    return _set(a, kw)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=0), dict(cols=96), dict(group=48), dict(dtype=3), dict(x=0),
                                 dict(weight=0), dict(codes=0), dict(scales=0), dict(delta=P), dict(weight=P + 8),
                                 dict(delta=P, sum=P + 8), dict(x_stride=257), dict(eps=-1.0), dict(eps=float("nan")),
                                 dict(cols=65536), dict(rows=1 << 31)], ids=str)
def test_norm_refuses(bad):
    lib = _lib.load()
    assert lib.ikl_add_rms_norm_int8(ctypes.byref(_norm(**bad)), None) in (_lib.IKL_EINVAL, _lib.IKL_EUNSUPPORTED)
    assert "rms norm int8" in _lib.last_error()


@pytest.mark.parametrize("bad", [(0, P, P, 4, 64, 64, 1), (P, 0, P, 4, 64, 64, 1), (P, P, 0, 4, 64, 64, 1),
                                 (P + 1, P, P, 4, 64, 64, 1), (P, P, P + 2, 4, 64, 64, 1), (P, P, P, -1, 64, 64, 1),
                                 (P, P, P, 4, 32, 64, 1), (P, P, P, 4, 64, 8, 1), (P, P, P, 4, 64, 64, 3),
                                 (P, P, P, 1 << 40, 64, 64, 1)], ids=str)
def test_dequantize_refuses(bad):
    codes, scales, out, rows, cols, group, dtype = bad
    lib = _lib.load()
    got = lib.ikl_dequantize_rows_int8(codes, scales, out, rows, cols, group, dtype, None)
    assert got in (_lib.IKL_EINVAL, _lib.IKL_EUNSUPPORTED) and "dequantize rows" in _lib.last_error()


def _linear(**kw):
    a = _lib.Int4LinearArgs()
    a.x = a.codes = a.scales = a.y = P
    a.rows, a.cols, a.out_cols, a.x_stride, a.y_stride = 4, 256, 48, 256, 48
    a.group, a.dtype = 64, _lib.IKL_BF16
    return _set(a, kw)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=0), dict(out_cols=0), dict(cols=96), dict(group=256),
                                 dict(dtype=3), dict(dtype=_lib.IKL_F32), dict(x=0), dict(codes=0), dict(scales=0),
                                 dict(y=0), dict(x=P + 8), dict(x_stride=12), dict(codes=P + 4), dict(scales=P + 4),
                                 dict(zeros=P + 2), dict(y=P + 1), dict(residual=P + 1), dict(gated=1, residual=P),
                                 dict(x_scales=P + 2), dict(rows=1 << 40), dict(cols=1 << 25), dict(out_cols=1 << 25)],
                         ids=str)
def test_linear_refuses(bad):
    lib = _lib.load()
    assert lib.ikl_int4_linear(ctypes.byref(_linear(**bad)), None) in (_lib.IKL_EINVAL, _lib.IKL_EUNSUPPORTED)
    assert "int4 linear" in _lib.last_error()


def test_no_rows_and_no_arguments():
    lib = _lib.load()
    for call, args in ((lib.ikl_quantize_rows_int8, _rows), (lib.ikl_add_rms_norm_int8, _norm),
                       (lib.ikl_int4_linear, _linear)):
        assert call(None, None) == _lib.IKL_EINVAL
        assert call(ctypes.byref(args(rows=0, x=0, codes=0)), None) == _lib.IKL_OK
    assert lib.ikl_dequantize_rows_int8(None, None, None, 0, 64, 64, 1, None) == _lib.IKL_OK
    assert lib.ikl_int4_linear_workspace_size(None) < 0
    assert lib.ikl_int4_linear_workspace_size(ctypes.byref(_linear(cols=96))) < 0
    assert lib.ikl_int4_linear_workspace_size(ctypes.byref(_linear())) >= 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("out,groups", [(2, 1), (16, 3), (34, 4), (96, 5)])
def test_packed_weights_hold_their_codes(group, gated, out, groups):
    gen = torch.Generator().manual_seed(out)
    codes = torch.randint(0, 16, (out, group * groups), generator=gen)
    scales = torch.rand(out, groups, generator=gen)
    zeros = torch.randint(0, 16, (out, groups), generator=gen)
    for z in (None, zeros):
        w = pack_int4_weight(codes, scales, z, group_size=group, gated=gated)
        grouped = codes.view(out, groups, group) - (8 if z is None else z[..., None])
        assert torch.equal(w.dequantize(), (grouped * scales[..., None]).view(out, -1))
        assert w.out_features == out // (1 + gated) and w.in_features == group * groups
        # rows past the last weigh nothing
        assert float(w.scales.abs().sum()) == pytest.approx(float(scales.sum()))


def test_layout_of_a_step():
    """Lane l, dword i, code j of the header's layout."""
    codes = torch.arange(16 * 256).view(16, 256) * 7 % 16
    for group in (32, 64, 128):
        w = pack_int4_weight(codes, torch.ones(16, 256 // group), group_size=group)
        for step, lane, i, j in ((0, 0, 0, 0), (1, 63, 3, 7), (0, 37, 2, 5), (1, 20, 1, 3)):
            q, r = lane // 16, lane % 16
            k = 128 * step + (32 * i + 8 * q if group == 32 else 64 * (i // 2) + 16 * q + 8 * (i % 2)) + j
            byte = int(w.codes[0, step, lane, 4 * i + j % 4])
            assert (byte >> (4 * (j // 4))) & 15 == int(codes[r, k])


def test_weights_refuse():
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1)
    for bad in (dict(codes=codes.float()), dict(codes=codes[0]), dict(codes=codes + 16), dict(codes=codes.int() - 1),
                dict(codes=codes[:, :48]), dict(scales=scales[:3]), dict(scales=scales.int()),
                dict(zeros=torch.full((4, 1), 16)), dict(zeros=scales), dict(zeros=torch.zeros(4, 2, dtype=torch.int)),
                dict(group_size=16), dict(codes=codes[:3], scales=scales[:3], gated=True),
                dict(codes=codes[:0], scales=scales[:0])):
        given = dict(codes=codes, scales=scales, zeros=None, group_size=64) | bad
        with pytest.raises(ValueError):
            pack_int4_weight(given.pop("codes"), given.pop("scales"), given.pop("zeros"), **given)
    for bad in (torch.ones(64), torch.ones(4, 64).double(), torch.full((4, 64), float("nan")), torch.ones(4, 60)):
        with pytest.raises(ValueError):
            quantize_int4_weight(bad, group_size=64)


def test_rows_in_8_bits_refuse():
    codes, scales = torch.zeros(3, 128, dtype=torch.int8), torch.ones(3, 2)
    rows = Int8Rows(codes, scales, 64)
    assert rows.shape == (3, 128) and rows.dtype == torch.bfloat16
    for bad in (dict(codes=codes.int()), dict(scales=scales.double()), dict(scales=scales[:2]), dict(group_size=128),
                dict(group_size=16), dict(codes=codes[0], scales=scales[0]), dict(dtype=torch.int8)):
        given = dict(codes=codes, scales=scales, group_size=64) | bad
        with pytest.raises(ValueError):
            Int8Rows(given.pop("codes"), given.pop("scales"), **given)


def test_a_weight_moves_whole():
    w = quantize_int4_weight(torch.randn(8, 64), group_size=32, symmetric=False)
    assert isinstance(w.to("cpu"), Int4Weight) and torch.equal(w.to("cpu").dequantize(), w.dequantize())
    assert w.nbytes == w.codes.numel() + 4 * w.scales.numel() + w.zeros.numel()
