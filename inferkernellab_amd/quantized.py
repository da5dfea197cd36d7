"""A layer's quantised work around the paged attention (csrc/int8_rows.hip,
csrc/int4_linear.hip): linear layers over 4-bit weights, and the rows in
8 bits that they take where the matrix cores bound them. The reference has no
quantised layers.

A weight ``W[n, k] = scale[n, g] * (code[n, k] - zero[n, g])`` has codes and
zero points of 0 to 15 and a scale for each output column ``n`` and group ``g``
of ``group_size`` (32, 64 or 128) entries of the contraction
(:class:`Int4Weight`). It is laid out once, by :func:`pack_int4_weight` or
:func:`quantize_int4_weight`.

Rows in 8 bits (:class:`Int8Rows`) have codes of -127 to 127 and a scale for
each row and group of columns, the group's largest magnitude over 127. They
come from :func:`quantize_rows_int8_hip`, :func:`add_rms_norm_int8_hip` and
:func:`silu_mul_int8_hip`; a group with a NaN or an infinity stands for NaN.

:func:`int4_linear_hip` multiplies 16-bit rows or rows in 8 bits with such a
weight: sums are fp32 (of 8-bit rows exact within a group) and rounded once,
with the residual's addition or ``SiLU(gate) * up`` before it. These operators
compute no gradients.

Each operator has a prepared form that checks its tensors once; its bound
tensors may be updated in place between calls. A prepared launch owns its
results and workspace: calls that may overlap need one each.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _DTYPES, _require_backend

GROUP_SIZES = (32, 64, 128)


def _launch(device: torch.device, call, *args) -> int:
    """`call(*args, stream)` on the current stream of `device` (of a tensor,
    so that torch has a GPU and the device an index)."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        return call(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(device):
        return call(*args, torch._C._cuda_getCurrentRawStream(index))


def _check_group(group_size: int, cols: int) -> None:
    if group_size not in GROUP_SIZES:
        raise ValueError("group_size must be 32, 64 or 128")
    if cols <= 0 or cols % group_size:
        raise ValueError(f"columns ({cols}) must be whole groups of {group_size}")


def _rows_of(x: torch.Tensor, name: str) -> torch.Tensor:
    """`x` as [rows, cols] whose rows can be read in 16-byte pieces, a copy
    where its own cannot."""
    if x.ndim < 2:
        raise ValueError(f"{name} must have shape [..., columns] with at least two dimensions")
    if x.device.type != "cuda":
        raise ValueError(f"{name} must be on a GPU (torch 'cuda' device)")
    flat = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    fits = (flat.shape[1] <= 1 or flat.stride(1) == 1) and flat.data_ptr() % 16 == 0 and (
        flat.shape[0] <= 1 or flat.stride(0) * flat.element_size() % 16 == 0)
    return flat if fits else flat.clone(memory_format=torch.contiguous_format)


def _check_like(x: torch.Tensor, y, name: str, shape=None) -> None:
    if not isinstance(y, torch.Tensor) or y.shape != (x.shape if shape is None else shape):
        raise ValueError(f"{name} must have shape {tuple(x.shape if shape is None else shape)}")
    if y.dtype != x.dtype or y.device != x.device:
        raise ValueError(f"{name} must have the rows' dtype and device")


def _apart(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether no byte of the rows [rows, columns] of `x` is one of `y`'s."""
    if not x.numel() or not y.numel():
        return True
    (x0, xs, xw), (y0, ys, yw) = ((t.data_ptr(), t.stride(0) * t.element_size(), t.shape[1] * t.element_size())
                                  for t in (x, y))
    if x0 + xs * (x.shape[0] - 1) + xw <= y0 or y0 + ys * (y.shape[0] - 1) + yw <= x0:
        return True
    # column ranges of one buffer
    return xs == ys > 0 and xw <= (y0 - x0) % xs <= xs - yw


# ------------------------------------------------------------- rows in 8 bits
class Int8Rows:
    """Rows in 8 bits: ``codes`` ``[..., columns]`` int8, ``scales``
    ``[..., columns / group_size]`` float32; ``dtype`` is that of the rows
    they came from. Contiguous ones, the codes 16-byte aligned, are held
    themselves, others as copies: the attributes are what a product reads."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, group_size: int = 128, *,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        if codes.dtype != torch.int8 or scales.dtype != torch.float32:
            raise ValueError("codes must be int8 and scales float32")
        if codes.ndim < 2:
            raise ValueError("codes must have shape [..., columns] with at least two dimensions")
        _check_group(group_size, codes.shape[-1])
        if scales.shape != (*codes.shape[:-1], codes.shape[-1] // group_size):
            raise ValueError("scales must have one entry per row and group of columns")
        if scales.device != codes.device:
            raise ValueError("scales must be on the codes' device")
        if dtype not in _DTYPES:
            raise ValueError("dtype must be float16, bfloat16 or float32")
        codes = codes if codes.is_contiguous() and codes.data_ptr() % 16 == 0 else codes.clone(
            memory_format=torch.contiguous_format)
        self._hold(codes, scales.contiguous(), group_size, dtype)

    @classmethod
    def empty(cls, shape, group_size: int, dtype: torch.dtype, device: torch.device) -> "Int8Rows":
        rows = cls.__new__(cls)
        rows._hold(torch.empty(shape, dtype=torch.int8, device=device),
                   torch.empty((*shape[:-1], shape[-1] // group_size), dtype=torch.float32, device=device),
                   group_size, dtype)
        return rows

    def _hold(self, codes, scales, group_size, dtype) -> None:
        self._codes, self._scales, self.group_size, self.dtype = codes, scales, group_size, dtype
        self.shape, self.device = codes.shape, codes.device
        cols = codes.shape[-1]
        self._read = (codes.data_ptr(), scales.data_ptr())
        self._sizes = (codes.numel() // cols, cols, group_size)

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    def dequantize(self, dtype: torch.dtype | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """What the codes stand for, in ``dtype`` (the rows' own), rounded once."""
        if self.device.type != "cuda":
            raise ValueError("rows must be on a GPU (torch 'cuda' device)")
        if out is None:
            dtype = self.dtype if dtype is None else dtype
            if dtype not in _DTYPES:
                raise ValueError("dtype must be float16, bfloat16 or float32")
            out = torch.empty(self.shape, dtype=dtype, device=self.device)
        elif (out.shape != self.shape or out.device != self.device or out.dtype not in _DTYPES
              or not out.is_contiguous() or dtype not in (None, out.dtype)):
            raise ValueError("out must be contiguous float16, bfloat16 or float32 with the rows' shape and device")
        lib = _lib._lib or _require_backend()
        status = _launch(self.device, lib.ikl_dequantize_rows_int8, *self._read, out.data_ptr(), *self._sizes,
                         _DTYPES[out.dtype])
        if status:
            _lib.check(status, "dequantize rows")
        return out


class _Prepared:
    """A bound launch: calls `_run(args, stream)` and returns `_out`."""

    def _bind(self, run, args, device, keep, out, what) -> None:
        self._run, self._args, self.device, self._keep, self._out, self._what = run, args, device, keep, out, what
        self._ref = ctypes.byref(args)

    def __call__(self):
        status = _launch(self.device, self._run, self._ref)
        if status:
            _lib.check(status, self._what)
        return self._out


def _no_copies(given, bound) -> None:
    for x, y in zip(given, bound):
        if x is not None and x.data_ptr() != y.data_ptr():
            raise ValueError("rows of a prepared launch must be contiguous and 16-byte aligned")


class PreparedQuantizeRowsInt8(_Prepared):
    """:func:`quantize_rows_int8_hip` checked once on a fixed tensor."""

    def __init__(self, x: torch.Tensor, *, group_size: int = 128):
        self._prepare(x, None, group_size)
        _no_copies((x,), self._keep)

    def _prepare(self, x, up, group_size) -> None:
        lib = _require_backend()
        if x.dtype not in _DTYPES:
            raise ValueError("rows must be float16, bfloat16 or float32")
        flat = _rows_of(x, "rows")
        _check_group(group_size, x.shape[-1])
        rows = Int8Rows.empty(x.shape, group_size, x.dtype, x.device)
        a = _lib.Int8RowsArgs()
        a.x, a.x_stride = flat.data_ptr(), flat.stride(0)
        keep = [flat]
        if up is not None:
            _check_like(x, up, "up")
            other = _rows_of(up, "up")
            a.up, a.up_stride = other.data_ptr(), other.stride(0)
            keep.append(other)
        a.codes, a.scales = rows.codes.data_ptr(), rows.scales.data_ptr()
        a.rows, a.cols = flat.shape
        a.group, a.dtype = group_size, _DTYPES[x.dtype]
        self._bind(lib.ikl_quantize_rows_int8, a, x.device, keep, rows, "int8 rows")


class PreparedSiluMulInt8(PreparedQuantizeRowsInt8):
    """:func:`silu_mul_int8_hip` checked once on fixed tensors."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, *, group_size: int = 128):
        self._prepare(gate, up, group_size)
        _no_copies((gate, up), self._keep)


class PreparedAddRMSNormInt8(_Prepared):
    """:func:`add_rms_norm_int8_hip` checked once on fixed tensors."""

    def __init__(self, x: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, *, eps: float = 1e-6,
                 group_size: int = 128):
        self._prepare(x, delta, weight, eps, group_size)
        _no_copies((x, weight) if delta is None else (x, weight, delta), self._keep)

    def _prepare(self, x, delta, weight, eps, group_size) -> None:
        lib = _require_backend()
        if x.dtype not in _DTYPES:
            raise ValueError("rows must be float16, bfloat16 or float32")
        flat = _rows_of(x, "x")
        _check_group(group_size, x.shape[-1])
        _check_like(x, weight, "weight", (x.shape[-1],))
        if not eps >= 0:
            raise ValueError("eps must be non-negative")
        gain = weight if weight.is_contiguous() and weight.data_ptr() % 16 == 0 else weight.clone(
            memory_format=torch.contiguous_format)
        rows = Int8Rows.empty(x.shape, group_size, x.dtype, x.device)
        a = _lib.NormInt8Args()
        a.x, a.x_stride, a.weight = flat.data_ptr(), flat.stride(0), gain.data_ptr()
        keep, total = [flat, gain], x
        if delta is not None:
            _check_like(x, delta, "delta")
            other = _rows_of(delta, "delta")
            total = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            a.delta, a.delta_stride, a.sum, a.sum_stride = (other.data_ptr(), other.stride(0), total.data_ptr(),
                                                            x.shape[-1])
            keep.append(other)
        a.codes, a.scales = rows.codes.data_ptr(), rows.scales.data_ptr()
        a.rows, a.cols = flat.shape
        a.group, a.dtype, a.eps = group_size, _DTYPES[x.dtype], eps
        self._bind(lib.ikl_add_rms_norm_int8, a, x.device, keep, (total, rows), "rms norm int8")


def quantize_rows_int8_hip(x: torch.Tensor, *, group_size: int = 128) -> Int8Rows:
    """Rows ``x`` ``[..., columns]`` (fp16, bf16, fp32) in 8 bits."""
    call = PreparedQuantizeRowsInt8.__new__(PreparedQuantizeRowsInt8)
    call._prepare(x, None, group_size)
    return call()


def silu_mul_int8_hip(gate: torch.Tensor, up: torch.Tensor, *, group_size: int = 128) -> Int8Rows:
    """``SiLU(gate) * up`` in 8 bits, fp32 up to its codes. Both may be column
    ranges of one tensor."""
    call = PreparedSiluMulInt8.__new__(PreparedSiluMulInt8)
    call._prepare(gate, up, group_size)
    return call()


def add_rms_norm_int8_hip(x: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, *, eps: float = 1e-6,
                          group_size: int = 128):
    """``(x + delta, the RMSNorm of it times weight in 8 bits)``; ``(x, ...)``
    without ``delta``. The sum is rounded to the rows' dtype, its norm is fp32
    up to its codes."""
    call = PreparedAddRMSNormInt8.__new__(PreparedAddRMSNormInt8)
    call._prepare(x, delta, weight, eps, group_size)
    return call()


# ------------------------------------------------------------- 4-bit weights
class Int4Weight:
    """A weight ``[out_features, in_features]`` in 4 bits, in the kernels'
    layout (include/ikl_paged.h, ikl_int4_linear). ``gated``: a gate's rows and
    an up projection's in turn, ``out_features`` of each; products with it are
    ``SiLU(gate) * up``."""

    def __init__(self, codes, scales, zeros, out_features, in_features, group_size, gated, dtype) -> None:
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.out_features, self.in_features, self.group_size = out_features, in_features, group_size
        self.gated, self.dtype = gated, dtype

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.zeros) if t is not None)

    def to(self, device) -> "Int4Weight":
        moved = (None if t is None else t.to(device) for t in (self.codes, self.scales, self.zeros))
        return Int4Weight(*moved, self.out_features, self.in_features, self.group_size, self.gated, self.dtype)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """``[out_features, in_features]`` (gated: the gate's rows, then the up
        projection's), rounded once from float32."""
        tiles, steps = self.codes.shape[:2]
        # [tile, step, q, row, dword, byte, half of byte]
        c = self.codes.view(tiles, steps, 4, 16, 4, 4)
        c = torch.stack((c & 15, c >> 4), -1).transpose(-1, -2)  # code 4 * half + byte of its dword
        if self.group_size == 32:  # k = 32 dword + 8 q + code
            c = c.permute(0, 3, 1, 4, 2, 5, 6)
        else:  # k = 64 (dword / 2) + 16 q + 8 (dword % 2) + code
            c = c.reshape(tiles, steps, 4, 16, 2, 2, 2, 4).permute(0, 3, 1, 4, 2, 5, 6, 7)
        c = c.reshape(tiles, 16, -1, self.group_size).float()
        zeros = 8.0 if self.zeros is None else self.zeros.transpose(1, 2).float()[..., None]
        w = ((c - zeros) * self.scales.transpose(1, 2)[..., None]).reshape(tiles, 16, -1)
        if self.gated:
            w = w.view(tiles // 2, 2, 16, -1).transpose(0, 1)
        w = w.reshape(2 if self.gated else 1, -1, w.shape[-1])[:, :self.out_features, :self.in_features]
        return w.reshape(-1, self.in_features).to(dtype)


def _padded(t: torch.Tensor, dim: int, to: int, value) -> torch.Tensor:
    if t.shape[dim] == to:
        return t
    shape = list(t.shape)
    shape[dim] = to - t.shape[dim]
    return torch.cat((t, t.new_full(shape, value)), dim)


def pack_int4_weight(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
                     group_size: int = 128, gated: bool = False) -> Int4Weight:
    """Lays a 4-bit weight out for the kernels, on its own device.

    ``codes`` ``[out, in]`` of whole numbers 0 to 15; ``scales``
    ``[out, in / group_size]`` floating; ``zeros`` like the scales, whole
    numbers 0 to 15 (8 where there are none). ``gated``: the rows are a gate's,
    then as many of an up projection's.
    """
    if codes.ndim != 2 or codes.dtype.is_floating_point or codes.dtype.is_complex or codes.dtype == torch.bool:
        raise ValueError("codes must be whole numbers with shape [out, in]")
    out, cols = codes.shape
    _check_group(group_size, cols)
    if out == 0 or (gated and out % 2):
        raise ValueError("a weight needs rows, a gated one an even number of them")
    groups = cols // group_size
    if scales.shape != (out, groups) or not scales.dtype.is_floating_point or scales.device != codes.device:
        raise ValueError("scales must be floating with one entry per row and group, on the codes' device")
    if zeros is not None and (zeros.shape != (out, groups) or zeros.dtype.is_floating_point
                              or zeros.device != codes.device):
        raise ValueError("zeros must be whole numbers with one entry per row and group, on the codes' device")
    for name, t in (("codes", codes), ("zeros", zeros)):
        if t is not None and (int(t.min()) < 0 or int(t.max()) > 15):
            raise ValueError(f"{name} must lie in 0 to 15")
    parts, per_step = 2 if gated else 1, 128 // group_size
    steps, tiles = -(-cols // 128), -(-(out // parts) // 16)

    def tiled(t, width, value):
        """[tiles (gate's and up's in turn), 16, width]"""
        t = _padded(_padded(t.view(parts, out // parts, -1), 1, 16 * tiles, value), 2, width, value)
        return t.view(parts, tiles, 16, width).transpose(0, 1).reshape(parts * tiles, 16, width)

    c = tiled(codes.to(torch.uint8).contiguous(), 128 * steps, 8)
    if group_size == 32:  # [tile, row, step, dword, q, half of byte, byte]
        c = c.view(-1, 16, steps, 4, 4, 2, 4).permute(0, 2, 4, 1, 3, 6, 5)
    else:  # [tile, row, step, dword / 2, q, dword % 2, half of byte, byte]
        c = c.view(-1, 16, steps, 2, 4, 2, 2, 4).permute(0, 2, 4, 1, 3, 5, 7, 6)
    c = (c[..., 0] | (c[..., 1] << 4)).reshape(parts * tiles, steps, 64, 16).contiguous()

    def laid_out(t, value):
        # a clone: of a contraction of one step all that is before it may be the caller's own memory
        return tiled(t.contiguous(), steps * per_step, value).transpose(1, 2).clone(
            memory_format=torch.contiguous_format)

    s = laid_out(scales.to(torch.float32), 0.0)
    z = None if zeros is None else laid_out(zeros.to(torch.uint8), 8)
    dtype = scales.dtype if scales.dtype in _DTYPES else torch.float32
    return Int4Weight(c, s, z, out // parts, cols, group_size, gated, dtype)


def quantize_int4_weight(weight: torch.Tensor, *, group_size: int = 128, symmetric: bool = True,
                         gated: bool = False) -> Int4Weight:
    """``weight`` ``[out, in]`` rounded to 4 bits, each group by its own range.

    ``symmetric``: steps of the largest magnitude over 7 around a zero of 8;
    else 15 steps from the smallest value (at most 0) to the largest (at least
    0). Steps are held in the weight's dtype, codes are the nearest.
    """
    if weight.ndim != 2 or weight.dtype not in _DTYPES:
        raise ValueError("weight must be float16, bfloat16 or float32 with shape [out, in]")
    _check_group(group_size, weight.shape[1])
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("weight must be finite")
    w = weight.detach().float().reshape(weight.shape[0], -1, group_size)
    if symmetric:
        low, span = None, w.abs().amax(-1) / 7
    else:
        low = w.amin(-1).clamp(max=0)
        high = w.amax(-1).clamp(min=0)
        span = (high - low) / 15
        span = torch.where(span.isfinite(), span, high / 15 - low / 15)  # a range past fp32's largest value
    # A zero group divides by its step too. A step below fp16's normal numbers may
    # have been rounded down by more than the codes' range has to spare.
    least = torch.finfo(weight.dtype).smallest_normal if weight.dtype != torch.float16 else 2.0 ** -24
    scales = span.to(weight.dtype).clamp(min=least)
    scales = torch.where(scales.float() * (1 + 2.0 ** -6) < span, scales * 2, scales)
    step = scales.float()
    zeros = None if low is None else (-low / step).round_().clamp_(0, 15)
    codes = (w / step[..., None] + (8.0 if zeros is None else zeros[..., None])).round_().clamp_(0, 15)
    return pack_int4_weight(codes.to(torch.uint8).view(weight.shape), scales,
                            None if zeros is None else zeros.to(torch.uint8), group_size=group_size, gated=gated)


class PreparedInt4Linear(_Prepared):
    """:func:`int4_linear_hip` checked once on fixed tensors."""

    def __init__(self, x, weight: Int4Weight, *, residual: torch.Tensor | None = None,
                 out: torch.Tensor | None = None):
        self._prepare(x, weight, residual, out)
        _no_copies((x.codes if isinstance(x, Int8Rows) else x, residual), self._keep)

    def _prepare(self, x, weight, residual, out) -> None:
        lib = _require_backend()
        if not isinstance(weight, Int4Weight):
            raise ValueError("weight must be an Int4Weight")
        a, scales = _lib.Int4LinearArgs(), None
        if isinstance(x, Int8Rows):
            if x.group_size != weight.group_size:
                raise ValueError("rows and weight must have the same group_size")
            flat = x.codes
            if flat.device.type != "cuda":
                raise ValueError("rows must be on a GPU (torch 'cuda' device)")
            a.x_scales = x.scales.data_ptr()
            flat, scales = flat.view(-1, flat.shape[-1]), x.scales.view(-1, x.scales.shape[-1])
        else:
            if x.dtype not in (torch.float16, torch.bfloat16):
                raise ValueError("rows must be float16, bfloat16 or Int8Rows")
            flat = _rows_of(x, "rows")
            a.x_stride = flat.stride(0)
        if x.shape[-1] != weight.in_features:
            raise ValueError(f"rows have {x.shape[-1]} columns, the weight takes {weight.in_features}")
        if weight.device != x.device:
            raise ValueError("weight must be on the rows' device")
        shape, given = (*x.shape[:-1], weight.out_features), out is not None
        if out is None:
            out = torch.empty(shape, dtype=x.dtype, device=x.device)
        elif out.shape != shape or out.dtype != x.dtype or out.device != x.device:
            raise ValueError(f"out must have shape {shape} and the rows' dtype and device")
        if out.ndim != 2 and not out.is_contiguous():
            raise ValueError("out of more than two dimensions must be contiguous")
        y = out if out.ndim == 2 else out.view(-1, weight.out_features)
        if y.shape[1] > 1 and y.stride(1) != 1:
            raise ValueError("out must be contiguous in its rows")
        if given and not (_apart(flat, y) and (scales is None or _apart(scales, y))):
            raise ValueError("out must not share memory with the rows")
        a.x, a.y, a.y_stride = flat.data_ptr(), y.data_ptr(), y.stride(0)
        keep = [flat, None, weight, x]
        if residual is not None:
            if weight.gated:
                raise ValueError("a gated weight takes no residual")
            if residual.shape != shape or residual.dtype != x.dtype or residual.device != x.device:
                raise ValueError(f"residual must have shape {shape} and the rows' dtype and device")
            keep[1] = r = residual if residual.ndim == 2 else residual.reshape(y.shape)
            if r.shape[1] > 1 and r.stride(1) != 1:
                keep[1] = r = r.contiguous()
            same = r.data_ptr() == y.data_ptr() and r.stride(0) == y.stride(0)
            if given and not same and not _apart(r, y):
                raise ValueError("out must be the residual or share no memory with it")
            a.residual, a.residual_stride = r.data_ptr(), r.stride(0)
        a.codes, a.scales = weight.codes.data_ptr(), weight.scales.data_ptr()
        a.zeros = None if weight.zeros is None else weight.zeros.data_ptr()
        a.rows, a.cols, a.out_cols = flat.shape[0], weight.in_features, weight.out_features
        a.group, a.gated, a.dtype = weight.group_size, weight.gated, _DTYPES[x.dtype]
        size = lib.ikl_int4_linear_workspace_size(ctypes.byref(a))
        if size:
            _lib.check(min(size, 0), "int4 linear")
            keep.append(torch.empty(size, dtype=torch.uint8, device=x.device))
            a.workspace, a.workspace_bytes = keep[-1].data_ptr(), size
        self._bind(lib.ikl_int4_linear, a, x.device, keep, out, "int4 linear")


def int4_linear_hip(x, weight: Int4Weight, *, residual: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """``x W^T`` over a 4-bit weight, ``[..., out_features]`` in ``x.dtype``.

    ``x``: fp16 or bf16 rows ``[..., in_features]``, or :class:`Int8Rows` of
    the weight's ``group_size``. ``residual`` (which may be ``out``) is added
    before the one rounding; a gated weight gives ``SiLU(gate) * up``. A row
    with a NaN or an infinity gives NaN or infinities.
    """
    call = PreparedInt4Linear.__new__(PreparedInt4Linear)
    call._prepare(x, weight, residual, out)
    return call()
