"""Rows in 8 bits and products with 4-bit weights against their definitions in
64 bits, from the same inputs.

Bounds. A rounding is off by at most half a step. An fp32 sum of n terms, each
addition rounded or cut to 24 bits, is off by at most (n - 1) 2^-23 of the
terms' magnitudes. 16-bit rows: a group's sum of x c and of x z, G terms each,
scaled and added to the other groups' (two more operations a group, and the
eight waves' sums): 2^-23 (G + 2 groups + 8) sum |x| s (c + z). 8-bit rows: the
group's sum P is exact, a is cut to 22 bits (3 2^-23 at most), a P rounds (half a
2^-23), then the multiply-adds with s over the groups and the eight waves' sums
(half each): 7.5 + groups / 2 of 2^-23, inside 2^-23 (groups + 2 + 8) sum over
groups |s a P|. Codes: what
they are rounded from is off by 127 times its relative error, in steps."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-23
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _half_step(want, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * want.abs() + f.eps * f.tiny / 2


def _weight(gen, outs, cols, group, *, zeros, gated=False, dtype=BF16):
    """(packed, [outs, cols] exact float64, |s| (c + z) of it)."""
    from inferkernellab_amd import pack_int4_weight

    c = torch.randint(0, 16, (outs, cols), generator=gen, device="cuda")
    s = ((torch.rand(outs, cols // group, generator=gen, device="cuda") + 0.5) * cols**-0.5 / 4).to(dtype)
    z = torch.randint(0, 16, s.shape, generator=gen, device="cuda") if zeros else None
    packed = pack_int4_weight(c.to(torch.uint8), s, None if z is None else z.to(torch.uint8), group_size=group,
                              gated=gated)
    z = torch.full_like(s, 8, dtype=torch.float64) if z is None else z.double()
    grouped, s = c.double().view(outs, -1, group), s.double()[..., None]
    return (packed, ((grouped - z[..., None]) * s).view(outs, cols), ((grouped + z[..., None]) * s).view(outs, cols))


def _mm(a, b):
    return torch.mm(a, b.t().contiguous())


def _expected(x, w, sums, residual, gated, dtype):
    """(value, bound) of a product with error `sums` before its epilogue."""
    y = _mm(x, w)
    if gated:
        half = y.shape[1] // 2
        g, u = y[:, :half], y[:, half:]
        dg, du = sums[:, :half], sums[:, half:]
        act = g * torch.sigmoid(g)
        # SiLU's slope is below 1.1; its exponential, sum and quotient and the
        # product round
        want = act * u
        return want, 1.1 * dg * (u.abs() + du) + act.abs() * du + 5 * U * want.abs() + _half_step(want, dtype)
    if residual is not None:
        want = y + residual.double()
        return want, sums + U * (y.abs() + want.abs()) + _half_step(want, dtype)
    return y, sums + _half_step(y, dtype)


def _assert_close(got, want, bound):
    assert got.shape == want.shape
    over = (got.double() - want).abs() - bound * (1 + 1e-9)
    assert bool((over <= 0).all()), (float(over.max()), float(want.abs().max()))


def _sums16(x, mag, group):
    groups = x.shape[1] // group
    return U * (group + 2 * groups + 8) * _mm(x.abs(), mag)


def _sums8(codes, scales, w, group):
    """The groups' sums by their magnitudes."""
    rows, groups = scales.shape
    total = torch.zeros(rows, w.shape[0], dtype=torch.float64, device="cuda")
    for g in range(groups):
        at = slice(g * group, (g + 1) * group)
        total += _mm(codes[:, at].double() * scales[:, g:g + 1].double(), w[:, at]).abs()
    return U * (groups + 10) * total


ROWS = [1, 5, 16, 17, 33, 64, 65, 130, 300]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("group,cols", [(32, 32), (32, 1184), (64, 192), (64, 1216), (128, 128), (128, 1408)])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_of_16_bit_rows(dtype, group, cols, zeros):
    from inferkernellab_amd import int4_linear_hip

    gen = _gen(cols + zeros)
    for outs, gated in ((16, False), (77, False), (272, False), (2 * 21, True), (2 * 160, True)):
        packed, w, mag = _weight(gen, outs, cols, group, zeros=zeros, gated=gated, dtype=dtype)
        assert torch.equal(packed.dequantize(torch.float32).double(), w.float().double())
        for rows in ROWS:
            x = torch.randn(rows, 2 * cols, generator=gen, device="cuda").to(dtype)[:, cols:]  # strided rows
            xd = x.double()
            sums = _sums16(xd, mag, group)
            want, bound = _expected(xd, w, sums, None, gated, dtype)
            _assert_close(int4_linear_hip(x, packed), want, bound)
            if not gated:
                res = torch.randn(rows, outs, generator=gen, device="cuda").to(dtype)
                want, bound = _expected(xd, w, sums, res, False, dtype)
                _assert_close(int4_linear_hip(x, packed, residual=res), want, bound)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("group,cols", [(32, 32), (32, 1184), (64, 192), (64, 1216), (128, 128), (128, 1408)])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_of_8_bit_rows(dtype, group, cols, zeros):
    from inferkernellab_amd import Int8Rows, int4_linear_hip

    gen = _gen(cols + zeros + 7)
    for outs, gated in ((16, False), (77, False), (272, False), (2 * 21, True), (2 * 160, True)):
        packed, w, _ = _weight(gen, outs, cols, group, zeros=zeros, gated=gated)
        for rows in ROWS:
            codes = torch.randint(-127, 128, (rows, cols), generator=gen, device="cuda").to(torch.int8)
            scales = torch.rand(rows, cols // group, generator=gen, device="cuda") / 60
            x = Int8Rows(codes, scales, group, dtype=dtype)
            xd = (codes.double().view(rows, -1, group) * scales.double()[..., None]).view(rows, cols)
            sums = _sums8(codes, scales, w, group)
            res = None if gated else torch.randn(rows, outs, generator=gen, device="cuda").to(dtype)
            want, bound = _expected(xd, w, sums, None, gated, dtype)
            _assert_close(int4_linear_hip(x, packed), want, bound)
            if not gated:
                want, bound = _expected(xd, w, sums, res, False, dtype)
                _assert_close(int4_linear_hip(x, packed, residual=res), want, bound)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("rows,outs,cols,group", [
    (16, 20000, 256, 64), (30, 9000, 384, 32), (130, 2070, 384, 128), (300, 2064, 640, 64), (100, 9000, 416, 32),
    (140, 4112, 3456, 128), (520, 2064, 3456, 64), (2050, 1040, 3456, 128), (520, 9000, 1408, 128),
    (700, 9000, 1376, 32), (6200, 5000, 320, 64), (6200, 4998, 384, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_larger_products(rows, outs, cols, group, zeros, eight):
    """Every form of a launch: blocks of 16 to 128 rows and 16 to 256 columns,
    contractions in one part and in several."""
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(rows + outs)
    gated = zeros and not eight
    packed, w, mag = _weight(gen, outs, cols, group, zeros=zeros, gated=gated)
    x = torch.randn(rows, cols, generator=gen, device="cuda").to(BF16)
    res = None if gated else torch.randn(rows, outs, generator=gen, device="cuda").to(BF16)
    if eight:
        x = quantize_rows_int8_hip(x, group_size=group)
        xd = (x.codes.double().view(rows, -1, group) * x.scales.double()[..., None]).view(rows, cols)
        sums = _sums8(x.codes, x.scales, w, group)
    else:
        xd = x.double()
        sums = _sums16(xd, mag, group)
    want, bound = _expected(xd, w, sums, res, gated, BF16)
    y = int4_linear_hip(x, packed, residual=res)
    _assert_close(y, want, bound)
    assert torch.equal(int4_linear_hip(x, packed, residual=res), y)


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_in_8_bits_up_to_the_largest_values(rows, zeros):
    """Whose products are finite."""
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(rows)
    packed, w, _ = _weight(gen, 80, 256, 128, zeros=zeros)
    packed.scales.mul_(2.0**-16)
    w = w * 2.0**-16
    x = torch.randn(rows, 256, generator=gen, device="cuda").clamp(-1, 1) * 2.0**127
    x[:, :2] = torch.finfo(FP32).max
    q = quantize_rows_int8_hip(x)
    xd = q.codes.double() * q.scales.double().repeat_interleave(128, 1)
    _assert_close(int4_linear_hip(q, packed), *_expected(xd, w, _sums8(q.codes, q.scales, w, 128), None, False, FP32))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("cols", [128, 256, 384, 512])
@pytest.mark.parametrize("rows", [300, 1900])
def test_short_contractions_over_many_rows(rows, cols, eight):
    """A workgroup's results pass through the memory that its last rows came
    into: each of many launches gives the same."""
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(cols + rows)
    packed, w, mag = _weight(gen, 4000, cols, 128, zeros=eight)
    x = torch.randn(rows, cols, generator=gen, device="cuda").to(BF16)
    q = quantize_rows_int8_hip(x)
    if eight:
        scales = q.scales.double().repeat_interleave(128, 1)
        xd, sums = q.codes.double() * scales, _sums8(q.codes, q.scales, w, 128)
    else:
        xd, sums = x.double(), _sums16(x.double(), mag, 128)
    first = int4_linear_hip(q if eight else x, packed)
    _assert_close(first, *_expected(xd, w, sums, None, False, BF16))
    for _ in range(20):
        assert torch.equal(int4_linear_hip(q if eight else x, packed), first)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("rows,cols", [(70000, 8192), (2200000, 32)])
def test_more_rows_than_a_grids_second_dimension_holds(rows, cols, eight):
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(11)
    packed, w, mag = _weight(gen, 16, cols, 32, zeros=False)
    x = torch.randn(rows, cols, generator=gen, device="cuda", dtype=BF16)
    given = quantize_rows_int8_hip(x, group_size=32) if eight else x
    y = int4_linear_hip(given, packed)
    part = slice(rows - 999, rows)  # and the rows before by themselves
    few = quantize_rows_int8_hip(x[part], group_size=32) if eight else x[part]
    xd = few.dequantize(FP32).double() if eight else few.double()
    # dequantised to fp32: half a step of each product more
    sums = _sums16(xd, mag, 32)
    want, bound = _expected(xd, w, sums, None, False, BF16)
    _assert_close(y[part], want, bound)
    for start in range(0, rows - 64, rows // 7):
        some = x[start:start + 64]
        if eight:
            some = quantize_rows_int8_hip(some, group_size=32).dequantize(FP32)
        want, bound = _expected(some.double(), w, _sums16(some.double(), mag, 32), None, False, BF16)
        _assert_close(y[start:start + 64], want, bound)


@pytest.mark.parametrize("rows", [3, 40, 200])
@pytest.mark.parametrize("eight", [False, True])
def test_nothing_outside_the_result_is_written(rows, eight):
    """Into columns 3 .. of a wider buffer with rows behind the last, in place
    of the residual, in leading dimensions."""
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(rows)
    packed, w, mag = _weight(gen, 45, 256, 64, zeros=True)
    x = torch.randn(rows, 256, generator=gen, device="cuda").to(BF16)
    given = quantize_rows_int8_hip(x, group_size=64) if eight else x
    wide = torch.full((rows + 20, 64), 7.0, dtype=BF16, device="cuda")
    wide[:rows, 3:48] = torch.randn(rows, 45, generator=gen, device="cuda").to(BF16)
    res = wide[:rows, 3:48].clone()
    out = wide[:rows, 3:48]
    assert int4_linear_hip(given, packed, residual=out, out=out) is out
    assert torch.equal(out, int4_linear_hip(given, packed, residual=res))
    wide[:rows, 3:48] = 7.0
    assert bool((wide == 7).all())
    folded = x.view(1, rows, 256)
    folded = quantize_rows_int8_hip(folded, group_size=64) if eight else folded
    y = int4_linear_hip(folded, packed, residual=res.view(1, rows, 45))
    assert y.shape == (1, rows, 45) and torch.equal(y[0], int4_linear_hip(given, packed, residual=res))


def test_empty_rows_give_empty_results():
    from inferkernellab_amd import add_rms_norm_int8_hip, int4_linear_hip, quantize_rows_int8_hip, silu_mul_int8_hip

    packed, _, _ = _weight(_gen(1), 48, 128, 128, zeros=False)
    x = torch.empty(0, 128, dtype=BF16, device="cuda")
    rows = quantize_rows_int8_hip(x)
    assert int4_linear_hip(x, packed).shape == (0, 48) and int4_linear_hip(rows, packed).shape == (0, 48)
    assert silu_mul_int8_hip(x, x).shape == (0, 128) and rows.dequantize().shape == (0, 128)
    total, rows = add_rms_norm_int8_hip(x, x, torch.ones(128, dtype=BF16, device="cuda"))
    assert total.shape == rows.shape == (0, 128)


@pytest.mark.parametrize("rows", [4, 100])
def test_a_row_that_is_not_finite_spoils_itself_alone(rows):
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(5)
    packed, _, _ = _weight(gen, 80, 256, 128, zeros=True)
    x = torch.randn(rows, 256, generator=gen, device="cuda").to(BF16)
    clean = int4_linear_hip(x, packed), int4_linear_hip(quantize_rows_int8_hip(x), packed)
    for value in (float("nan"), float("inf"), float("-inf")):
        bad = x.clone()
        bad[2, 130] = value
        codes = quantize_rows_int8_hip(bad)
        values = codes.dequantize()
        assert bool(values[2, 128:].isnan().all()) and bool(values[2, :128].isfinite().all())
        for y, fine in zip((int4_linear_hip(bad, packed), int4_linear_hip(codes, packed)), clean):
            assert not bool(y[2].isfinite().any())
            keep = [r for r in range(rows) if r != 2]
            assert torch.equal(y[keep], fine[keep])


# ------------------------------------------------------------ rows in 8 bits
def _check_codes(rows, values, error, dtype):
    """`values` float64 [rows, cols], off by at most `error` of themselves in fp32."""
    group = rows.group_size
    grouped = values.reshape(-1, values.shape[-1] // group, group)
    most = grouped.abs().amax(-1).clamp(min=2.0**-100)
    scales = rows.scales.double().view(most.shape)
    assert bool(((scales * 127 / most - 1).abs() <= error + 2.0**-24 * 1.01).all())
    codes = rows.codes.view(grouped.shape).double()
    assert int(codes.abs().max()) <= 127
    # the quotient: its dividend, the inverse scale's rounding and maximum
    off = (codes - grouped * 127 / most[..., None]).abs()
    assert float(off.max()) <= 0.5 + 127 * (2 * error + 2.0**-23), float(off.max())
    stand = codes * rows.scales.double().view(most.shape)[..., None]
    _assert_close(rows.dequantize().view(grouped.shape), stand, _half_step(stand, dtype))


SHAPES = [(1, 128), (3, 384), (17, 2048), (129, 4224), (5, 11264)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_in_8_bits(dtype, group):
    from inferkernellab_amd import quantize_rows_int8_hip, silu_mul_int8_hip

    for rows, cols in SHAPES:
        gen = _gen(rows + group)
        both = torch.randn(rows, 2 * cols, generator=gen, device="cuda").to(dtype)
        x, up = both[:, :cols], both[:, cols:]
        x[0, :group] = 0
        got = quantize_rows_int8_hip(x, group_size=group)
        _check_codes(got, x.double(), 0.0, dtype)
        assert int(got.codes[0, :group].abs().max()) == 0
        d = x.double()
        # the exponential to an ulp, its sum, quotient and the product
        _check_codes(silu_mul_int8_hip(x, up, group_size=group), d * torch.sigmoid(d) * up.double(), 5 * 2.0**-24 + U,
                     dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("add", [False, True])
def test_norm_in_8_bits(dtype, group, add):
    from inferkernellab_amd import add_rms_norm_int8_hip

    for rows, cols in SHAPES:
        gen = _gen(rows + group)
        x = torch.randn(rows, cols, generator=gen, device="cuda").to(dtype)
        delta = torch.randn(rows, 2 * cols, generator=gen, device="cuda").to(dtype)[:, :cols] if add else None
        w = (1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(dtype)
        total, got = add_rms_norm_int8_hip(x, delta, w, eps=1e-6, group_size=group)
        expected = x + delta if add else x
        assert torch.equal(total, expected)
        t = expected.double()
        v = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        # a thread's squares in a chain of up to 128, 9 levels and eps, halved
        # by the root; rsqrtf to an ulp; two products
        _check_codes(got, v, (128 + 10) / 2 * 2.0**-24 + U + 2 * 2.0**-24, dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_codes_of_normalised_16_bit_rows_are_the_nearest(dtype):
    """They depend on x times weight alone, exact in fp32; fp16's quotient by
    127 / amax is rounded once, 2^-16 of a step."""
    from inferkernellab_amd import add_rms_norm_int8_hip

    gen = _gen(6)
    x = torch.randn(513, 2048, generator=gen, device="cuda").to(dtype)
    w = (1 + 0.1 * torch.randn(2048, generator=gen, device="cuda")).to(dtype)
    _, got = add_rms_norm_int8_hip(x, None, w, group_size=32)
    g = (x.double() * w.double()).view(513, -1, 32)
    share = g * 127 / g.abs().amax(-1, keepdim=True)
    off = (got.codes.view_as(share).double() - share).abs()
    assert float(off.max()) <= 0.5 + (0 if dtype == BF16 else 2.0**-16)


def test_norms_of_rows_near_the_ends_of_fp32():
    """Groups far below their row, rows whose squares overflow (their norm is 0
    in fp32 arithmetic) and rows of zeros."""
    from inferkernellab_amd import add_rms_norm_int8_hip

    x = torch.zeros(5, 256, device="cuda")
    x[0, :128] = torch.linspace(-1e15, 1e15, 128, device="cuda")
    x[0, 128:] = torch.linspace(-1e-20, 1e-20, 128, device="cuda")
    x[1] = 1e30
    x[2] = torch.linspace(-1e-30, 1e-30, 256, device="cuda")
    x[3, 7] = float("nan")
    w = torch.ones(256, device="cuda")
    _, got = add_rms_norm_int8_hip(x, None, w, eps=1e-6)
    keep = torch.tensor([0, 2, 4], device="cuda")
    t = x[keep].double()
    v = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)
    from inferkernellab_amd import Int8Rows
    _check_codes(Int8Rows(got.codes[keep], got.scales[keep], 128, dtype=FP32), v, 74 * 2.0**-24 + U, FP32)
    values = got.dequantize()
    assert bool((values[1] == 0).all()) and bool(values[3].isnan().all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_norms_whose_products_without_the_rows_factor_leave_fp32(dtype):
    """x times weight past fp32's largest value or below its normal ones, their
    norms inside."""
    from inferkernellab_amd import add_rms_norm_int8_hip

    for size, gain in ((2.0**14, 2.0**119), (2.0**-60, 2.0**-80)):
        gen = _gen(9)
        x = (torch.randn(7, 256, generator=gen, device="cuda") * size).to(dtype)
        w = torch.ones(256, device="cuda")
        w[128:] = gain * (1 + torch.rand(128, generator=gen, device="cuda"))
        _, got = add_rms_norm_int8_hip(x, None, w.to(dtype), eps=0.0)
        t = x.double()
        v = t * torch.rsqrt(t.square().mean(-1, keepdim=True)) * w.to(dtype).double()
        assert float(v.abs().max()) < torch.finfo(dtype).max
        # as in test_norm_in_8_bits, of 256 columns: up to 8 squares a thread
        _check_codes(got, v, (8 + 10) / 2 * 2.0**-24 + U + 2 * 2.0**-24, dtype)


def test_norms_past_fp32_stand_for_nan():
    from inferkernellab_amd import add_rms_norm_int8_hip

    x = torch.ones(1, 256, device="cuda")
    x[0, 0] = 8.0  # its norm is 7.2 or so
    w = torch.ones(256, device="cuda")
    w[:128] = 2.0**126
    _, got = add_rms_norm_int8_hip(x, None, w, eps=0.0)
    values = got.dequantize()
    assert bool(values[0, :128].isnan().all()) and bool(values[0, 128:].isfinite().all())


def test_values_near_the_ends_of_fp32_keep_their_codes():
    from inferkernellab_amd import quantize_rows_int8_hip

    x = torch.zeros(5, 128, device="cuda")
    x[0] = torch.linspace(-3.4e38, 3.4e38, 128, dtype=torch.float64, device="cuda")  # its width is past fp32
    x[1] = torch.linspace(-(2.0**-99), 2.0**-99, 128, device="cuda")
    x[2] = 2.0**-140  # below a step of the smallest scale
    x[3] = torch.linspace(-127, 127, 128, device="cuda")
    got = quantize_rows_int8_hip(x)
    _check_codes(got, x.double(), 0.0, FP32)
    assert int(got.codes[2].abs().max()) == int(got.codes[4].abs().max()) == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_codes_of_16_bit_rows_are_the_nearest(dtype):
    """127 v / amax of 16-bit values lies on a half often, and otherwise 2^-16
    from one at least: 64 bits tell."""
    from inferkernellab_amd import quantize_rows_int8_hip

    x = torch.randn(513, 2048, generator=_gen(4), device="cuda").to(dtype)
    got = quantize_rows_int8_hip(x, group_size=32)
    g = x.double().view(513, -1, 32)
    share = g * 127 / g.abs().amax(-1, keepdim=True)
    assert bool((share.abs() % 1 == 0.5).any())
    assert torch.equal(got.codes.view_as(share), share.round().to(torch.int8))


def test_ties_go_to_the_even_code():
    from inferkernellab_amd import quantize_rows_int8_hip

    x = torch.zeros(1, 32, device="cuda")
    x[0, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5])
    assert quantize_rows_int8_hip(x, group_size=32).codes[0, :6].tolist() == [127, 0, 2, 2, 0, -2]


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("rows", [1, 29, 150])
@pytest.mark.parametrize("eight", [False, True])
def test_a_gated_mlp(rows, eight):
    """norm -> gate and up -> 8 bits -> down + residual, every stage against its
    definition on what the stage before it left."""
    from inferkernellab_amd import (add_rms_norm_int8_hip, int4_linear_hip, quantize_rows_int8_hip, silu_mul_int8_hip)

    gen = _gen(rows)
    hidden, inner, group = 512, 704, 64
    x, delta = torch.randn(2, rows, hidden, generator=gen, device="cuda").to(BF16)
    norm = (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).to(BF16)
    gate_up, wgu, mgu = _weight(gen, 2 * inner, hidden, group, zeros=True)
    down, wd, md = _weight(gen, hidden, inner, group, zeros=False)
    total, codes = add_rms_norm_int8_hip(x, delta, norm, group_size=group)
    if eight:
        both = int4_linear_hip(codes, gate_up)
        act = silu_mul_int8_hip(both[:, :inner], both[:, inner:], group_size=group)
        a = (act.codes.double().view(rows, -1, group) * act.scales.double()[..., None]).view(rows, inner)
        sums = _sums8(act.codes, act.scales, wd, group)
    else:
        both = int4_linear_hip(codes.dequantize(), gate_up)
        act = silu_mul_int8_hip(both[:, :inner], both[:, inner:], group_size=group).dequantize()
        a = act.double()
        sums = _sums16(a, md, group)
    want, bound = _expected(a, wd, sums, total, False, BF16)
    _assert_close(int4_linear_hip(act, down, residual=total), want, bound)
    # the gated weight of the same rows: one rounding less than the two steps
    fused = quantize_rows_int8_hip(x, group_size=group) if eight else x
    assert int4_linear_hip(fused, _gated(gate_up, inner)).shape == (rows, inner)


def _gated(w, inner):
    from inferkernellab_amd import quantize_int4_weight

    return quantize_int4_weight(w.dequantize(), group_size=w.group_size, gated=True)


# ------------------------------------------------- prepared, captured, streams
def _launches(gen, rows):
    """(prepared call, how to make its inputs anew) of each operator."""
    import inferkernellab_amd as ikl

    x, delta = torch.randn(2, rows, 256, generator=gen, device="cuda").to(BF16)
    norm = torch.ones(256, dtype=BF16, device="cuda")
    packed, _, _ = _weight(gen, 100, 256, 64, zeros=True)
    q = ikl.quantize_rows_int8_hip(x, group_size=64)
    res = torch.randn(rows, 100, generator=gen, device="cuda").to(BF16)
    return x, delta, [
        (ikl.PreparedInt4Linear(x, packed, residual=res), lambda: ikl.int4_linear_hip(x, packed, residual=res)),
        (ikl.PreparedInt4Linear(q, packed), lambda: ikl.int4_linear_hip(q, packed)),
        (ikl.PreparedQuantizeRowsInt8(x, group_size=64), lambda: ikl.quantize_rows_int8_hip(x, group_size=64)),
        (ikl.PreparedSiluMulInt8(x, delta, group_size=32), lambda: ikl.silu_mul_int8_hip(x, delta, group_size=32)),
        (ikl.PreparedAddRMSNormInt8(x, delta, norm), lambda: ikl.add_rms_norm_int8_hip(x, delta, norm)),
    ]


@pytest.mark.parametrize("rows", [40, 600])
def test_captured_eager_calls_hold_their_workspaces(rows):
    """Calls that split the contraction, in two graphs, replayed in turn with
    eager calls between."""
    import inferkernellab_amd as ikl

    gen = _gen(rows)
    packed, _, _ = _weight(gen, 2064, 3456, 64, zeros=True)
    x = torch.randn(rows, 3456, generator=gen, device="cuda").to(BF16)
    graphs = []
    ikl.int4_linear_hip(ikl.quantize_rows_int8_hip(x, group_size=64), packed)
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            q = ikl.quantize_rows_int8_hip(x, group_size=64)
            out = ikl.int4_linear_hip(x, packed), ikl.int4_linear_hip(q, packed)
        graphs.append((g, out))
    for _ in range(3):
        x.copy_(torch.randn(rows, 3456, generator=gen, device="cuda"))
        for g, out in graphs:
            g.replay()
            want = ikl.int4_linear_hip(x, packed), ikl.int4_linear_hip(ikl.quantize_rows_int8_hip(x, group_size=64),
                                                                       packed)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_results_that_share_memory_are_refused():
    from inferkernellab_amd import Int8Rows, int4_linear_hip

    packed, _, _ = _weight(_gen(1), 128, 128, 64, zeros=False)
    wide = torch.randn(5, 256, device="cuda").to(BF16)
    x = wide[:, :128]
    apart = int4_linear_hip(x, packed, out=wide[:, 128:])  # columns beside the rows
    assert torch.equal(apart, int4_linear_hip(x, packed))
    for out in (x, wide[:, 64:192]):
        with pytest.raises(ValueError, match="share"):
            int4_linear_hip(x, packed, out=out)
    other = torch.randn(5, 128, device="cuda").to(BF16)
    with pytest.raises(ValueError, match="residual"):
        int4_linear_hip(other, packed, residual=wide[:, :128], out=wide[:, 8:136])
    flat = torch.zeros(20 * 128, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        int4_linear_hip(other, packed, out=flat.as_strided((5, 128), (64, 1)))
    codes = torch.zeros(5, 128, dtype=torch.int8, device="cuda")
    rows = Int8Rows(codes, torch.ones(5, 2, device="cuda"), 64, dtype=BF16)
    half, _, _ = _weight(_gen(1), 64, 128, 64, zeros=False)
    with pytest.raises(ValueError, match="share"):
        int4_linear_hip(rows, half, out=codes.view(BF16))


def _parts(result):
    for r in result if isinstance(result, tuple) else (result,):
        yield from (r,) if isinstance(r, torch.Tensor) else (r.codes, r.scales)


@pytest.mark.parametrize("rows", [2, 70, 513])
def test_captured_launches_replay_the_eager_results(rows):
    gen = _gen(rows)
    x, delta, calls = _launches(gen, rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for prepared, _ in calls:
            prepared()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = [prepared() for prepared, _ in calls]
    for _ in range(3):
        x.copy_(torch.randn(rows, 256, generator=gen, device="cuda"))
        delta.copy_(torch.randn(rows, 256, generator=gen, device="cuda"))
        for r in results:
            for t in _parts(r):
                t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, (_, eager) in zip(results, calls):
            for a, b in zip(_parts(got), _parts(eager())):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    gen = _gen(3)
    jobs = [_launches(gen, rows)[2] for rows in (70, 513)]
    want = [[[t.clone() for t in _parts(eager())] for _, eager in calls] for calls in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, calls in zip(streams, jobs):
            with torch.cuda.stream(s):
                for prepared, _ in calls:
                    prepared()
    torch.cuda.synchronize()
    for calls, expected in zip(jobs, want):
        for (prepared, _), e in zip(calls, expected):
            assert all(torch.equal(a, b) for a, b in zip(_parts(prepared._out), e))


@pytest.mark.parametrize("rows", [3, 70])
def test_rows_past_32_bit_offsets(rows):
    """Rows 2^31 / (rows - 1) elements apart and more: offsets past 2^32 bytes."""
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(9)
    stride = (2**31 // (rows - 1) + 64) // 8 * 8
    packed, w, mag = _weight(gen, 80, 256, 64, zeros=False)
    far = torch.empty((rows - 1) * stride + 256, dtype=BF16, device="cuda").as_strided((rows, 256), (stride, 1))
    far.copy_(torch.randn(rows, 256, generator=gen, device="cuda"))
    near = far.contiguous()
    assert torch.equal(int4_linear_hip(far, packed), int4_linear_hip(near, packed))
    a, b = quantize_rows_int8_hip(far), quantize_rows_int8_hip(near)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    out = torch.empty((rows - 1) * stride + 80, dtype=BF16, device="cuda").as_strided((rows, 80), (stride, 1))
    assert torch.equal(int4_linear_hip(near, packed, out=out), int4_linear_hip(near, packed))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("symmetric", [False, True])
def test_quantized_weights(dtype, symmetric):
    """Half a step of each weight, the step rounded to the dtype; two codes'
    range is kept whole."""
    from inferkernellab_amd import quantize_int4_weight

    gen = _gen(2)
    w = torch.randn(70, 256, generator=gen, device="cuda").to(dtype)
    w[3] = 0
    w[4] = w[4].abs()
    q = quantize_int4_weight(w, group_size=64, symmetric=symmetric)
    g = w.double().view(70, -1, 64)
    if symmetric:
        step = g.abs().amax(-1, keepdim=True) / 7
    else:
        step = (g.amax(-1, keepdim=True).clamp(min=0) - g.amin(-1, keepdim=True).clamp(max=0)) / 15
    # the step's rounding moves a code by up to 15 of its steps; the zero point
    # is a whole number: another half step
    slack = 15 * torch.finfo(dtype).eps / 2 + 2.0**-20
    bound = step * ((0.5 if symmetric else 1.0) + slack) + torch.finfo(dtype).tiny
    assert bool(((q.dequantize(torch.float64).view_as(g) - g).abs() <= bound).all())
    assert torch.equal(q.dequantize()[3], torch.zeros(256, device="cuda"))
