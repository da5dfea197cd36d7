"""The quantised operators over the whole range of their types: gates far from
0, 16-bit rows up to their largest values, the mean of 8-bit rows' products.
Against the definitions in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-23
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
GATES = [-87.0, -87.5, -88.0, -88.5, -90.0, -95.0, -100.0, -103.0, -104.0, -110.0, -1e4, -6e4, -0.0, 0.0, 1e-30, -1e-30,
         0.5, -0.5, 17.0, -17.0, 87.0, 88.5, 110.0, 6e4]


def _silu(x):
    return x * torch.sigmoid(x)


def _silu_bound(x, up):
    """Of SiLU(x) * up in fp32: e^-x to an ulp of the power of two and what its
    argument's two products leave (each half a step of 2^-25, times ln 2: 0.17
    ulp together), its sum with 1 half an ulp, the reciprocal one, two products
    half an ulp each: 3.67. Below fp32's normal numbers the quotient, |x| times,
    and SiLU are off by half of 2^-149 each."""
    return 3.67 * U * (_silu(x) * up).abs() + (x.abs() + 1) * 2.0**-149 * up.abs()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_silu_in_8_bits_of_gates_far_from_0(dtype):
    """A group of equal values: its largest magnitude is any one's."""
    from inferkernellab_amd import silu_mul_int8_hip

    gates = GATES if dtype == FP16 else GATES + [-1e30, -3e38]
    x = torch.tensor(gates, dtype=torch.float64).to(dtype).cuda().view(-1, 1).expand(-1, 64).contiguous()
    for size in (1.0, 2.0**15 if dtype == FP16 else 2.0**100):
        up = torch.full_like(x, size)
        xd, ud = x.double(), up.double()
        got = silu_mul_int8_hip(x, up, group_size=32)
        stands = got.codes.double() * got.scales.double().repeat_interleave(32, 1)
        want = _silu(xd) * ud
        # the scale's rounding; values below half a step of the least scale are 0
        bound = _silu_bound(xd, ud) * (1 + 2.0**-20) + U / 2 * want.abs() + torch.where(
            want.abs() < 2.0**-100, 2.0**-100 / 254 * 1.01, 0.0)
        over = (stands - want).abs() - bound
        assert bool((over <= 0).all()), [(g, float(s[0]), float(w[0])) for g, s, w, o in zip(gates, stands, want, over)
                                         if float(o.max()) > 0]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_silu_in_8_bits_of_gates_that_are_not_finite(dtype):
    """SiLU of minus infinity is the product of an infinity and 0."""
    from inferkernellab_amd import silu_mul_int8_hip

    inf = float("inf")
    x = torch.ones(4, 64, device="cuda").to(dtype)
    x[0, 40], x[1, 40], x[2, 40] = inf, -inf, float("nan")
    values = silu_mul_int8_hip(x, torch.ones_like(x), group_size=32).dequantize()
    assert bool(values[:3, 32:].isnan().all()) and bool(values[:3, :32].isfinite().all())
    assert bool(values[3].isfinite().all())


@pytest.mark.parametrize("rows", [1, 400, 6200])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "8 bits to bf16", "8 bits to fp32"])
def test_gated_products_of_gates_far_from_0(kind, rows):
    """Each row has a gate and an up value of its own: the weight takes them from
    two entries of the contraction, in groups apart, times 1."""
    from inferkernellab_amd import Int8Rows, int4_linear_hip, pack_int4_weight

    outs, cols = (2048 if rows > 1000 else 40), 320
    codes = torch.full((2 * outs, cols), 8, dtype=torch.uint8)
    codes[:outs, 3], codes[outs:, 70] = 9, 9
    packed = pack_int4_weight(codes.cuda(), torch.ones(2 * outs, cols // 64, device="cuda"), group_size=64, gated=True)
    gates = torch.tensor(GATES if kind == "fp16" else GATES + [-1e30, 1e30], dtype=torch.float64)
    dtype = {"fp16": FP16, "8 bits to fp32": FP32}.get(kind, BF16)
    gate = gates[torch.arange(rows) % len(gates)].to(FP16 if kind == "fp16" else BF16).double().cuda()
    sizes = (1.0, 0.75, 2.0**6) if kind == "fp16" else (1.0, 0.75, 2.0**100)
    for size in sizes:
        # (finite results)
        up = torch.full_like(gate, size)
        up = torch.where(gate.abs() * up > torch.finfo(dtype).max, 1.0, up)
        if kind.startswith("8"):
            q = torch.zeros(rows, cols, dtype=torch.int8, device="cuda")
            q[:, 3], q[:, 70] = torch.where(gate < 0, -1, 1).to(torch.int8), 1
            scales = torch.ones(rows, cols // 64, device="cuda")
            scales[:, 0], scales[:, 1] = gate.abs(), up
            x = Int8Rows(q, scales, 64, dtype=dtype)
        else:
            x = torch.zeros(rows, cols, dtype=dtype, device="cuda")
            x[:, 3], x[:, 70] = gate.to(dtype), up.to(dtype)
        y = int4_linear_hip(x, packed).double()
        want = _silu(gate) * up
        f = torch.finfo(dtype)
        bound = _silu_bound(gate, up) * (1 + 2.0**-7) + f.eps / 2 * want.abs() + f.eps * f.tiny / 2
        over = (y - want[:, None]).abs().amax(1) - bound
        assert bool((over <= 0).all()), [(float(g), float(v), float(w)) for g, v, w, o in zip(gate, y[:, 0], want, over)
                                         if float(o) > 0][:8]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,outs,cols,group", [(3, 80, 256, 128), (16, 20000, 256, 64), (40, 2064, 384, 32),
                                                  (130, 2070, 384, 128), (300, 2064, 640, 64), (520, 9000, 384, 128),
                                                  (6200, 5000, 320, 64), (6200, 4998, 384, 128)])
def test_16_bit_rows_up_to_their_largest_values(rows, outs, cols, group, zeros, dtype):
    """Whose products are finite: group sums, with or without the zero point, are too."""
    from inferkernellab_amd import int4_linear_hip
    from tests.test_gpu_quantized import _assert_close, _expected, _gen, _sums16, _weight

    gen = _gen(rows + outs)
    packed, w, mag = _weight(gen, outs, cols, group, zeros=zeros, dtype=FP32)
    packed.scales.mul_(2.0**-16)
    w, mag = w * 2.0**-16, mag * 2.0**-16
    most = torch.finfo(dtype).max
    x = ((torch.rand(rows, cols, generator=gen, device="cuda", dtype=torch.float64) * 2 - 1) * most).to(dtype)
    x[0], x[1, ::2], x[1, 1::2], x[2] = most, most, -most, -most
    xd = x.double()
    want, bound = _expected(xd, w, _sums16(xd, mag, group), None, False, dtype)
    got = int4_linear_hip(x, packed)
    assert bool(got.isfinite().all())
    _assert_close(got, want, bound)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,outs", [(3, 80), (130, 2070), (6200, 5000)])
def test_16_bit_rows_below_the_normal_numbers(rows, outs, dtype):
    """Products of subnormal values with codes are kept, whatever power of two
    the codes are held at: of bf16 they are whole numbers of 2^-133 times 2^-11,
    below 2^24 of them in a group, so that nothing of them is rounded."""
    from inferkernellab_amd import int4_linear_hip
    from tests.test_gpu_quantized import _assert_close, _expected, _gen, _sums16, _weight

    f = torch.finfo(dtype)
    gen = _gen(rows)
    packed, w, mag = _weight(gen, outs, 320, 64, zeros=True, dtype=FP32)
    up = 2.0**100 if dtype == BF16 else 2.0**10
    packed.scales.mul_(up)
    w, mag = w * up, mag * up
    x = (torch.randint(-60, 61, (rows, 320), generator=gen, device="cuda").double() * f.tiny * f.eps).to(dtype)
    xd = x.double()
    want, bound = _expected(xd, w, _sums16(xd, mag, 64), None, False, dtype)
    _assert_close(int4_linear_hip(x, packed), want, bound)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,outs", [(16, 2048), (512, 2048), (6200, 4096)])
def test_products_of_8_bit_rows_are_not_shifted(rows, outs, zeros):
    """Terms of one sign: the relative error of y is the mean of its groups'. A
    scale of a row rounded to 22 bits is off by 0, 1, 2 and -1 quarters of a step
    of 2^-21, at most 1.23 2^-23 in the root mean square and 0 in the mean; so the mean over
    rows * groups of them stays within 6 of its standard deviations. The
    roundings behind it, more by the columns, add less than 0.01 2^-23 to that."""
    from inferkernellab_amd import Int8Rows, int4_linear_hip, pack_int4_weight
    from tests.test_gpu_quantized import _gen, _mm

    gen, cols, group = _gen(rows), 1024, 64
    codes = torch.randint(8, 16, (outs, cols), generator=gen, device="cuda").to(torch.uint8)
    z = torch.randint(0, 8, (outs, cols // group), generator=gen, device="cuda") if zeros else None
    packed = pack_int4_weight(codes, torch.rand(outs, cols // group, generator=gen, device="cuda") + 0.5, z,
                              group_size=group)
    q = torch.randint(1, 128, (rows, cols), generator=gen, device="cuda").to(torch.int8)
    scales = torch.rand(rows, cols // group, generator=gen, device="cuda") + 0.5
    xd = (q.double().view(rows, -1, group) * scales.double()[..., None]).view(rows, cols)
    want = _mm(xd, packed.dequantize(torch.float64))
    got = int4_linear_hip(Int8Rows(q, scales, group, dtype=FP32), packed).double()
    shift = float((got / want - 1).mean()) / U
    assert abs(shift) <= 6 * 1.23 / (rows * cols // group) ** 0.5 + 0.01, shift


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("zeros", [False, True])
def test_any_nan_or_infinity_as_the_scale_of_a_row(rows, zeros):
    """Of every bit pattern, the largest finite scales beside them."""
    from inferkernellab_amd import Int8Rows, int4_linear_hip
    from tests.test_gpu_quantized import _assert_close, _expected, _gen, _sums8, _weight

    gen = _gen(rows)
    packed, w, _ = _weight(gen, 80, 256, 64, zeros=zeros, dtype=FP32)
    packed.scales.mul_(2.0**-16)
    w = w * 2.0**-16
    q = torch.randint(-127, 128, (rows, 256), generator=gen, device="cuda").to(torch.int8)
    scales = torch.ones(rows, 4, device="cuda")
    scales[0, 1] = torch.finfo(FP32).max / 127
    for bits in (0x7F800000, -0x800000, 0x7F800001, 0x7FC00000, 0x7FFFFFFF, 0x7FFFFFFE, -1, -2, -0x400000):
        scales.view(torch.int32)[1, 2] = bits
        y = int4_linear_hip(Int8Rows(q, scales, 64, dtype=FP32), packed)
        assert not bool(y[1].isfinite().any()), hex(bits)
        keep = [r for r in range(rows) if r != 1]
        xd = q[keep].double() * scales[keep].double().repeat_interleave(64, 1)
        _assert_close(y[keep], *_expected(xd, w, _sums8(q[keep], scales[keep], w, 64), None, False, FP32))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_a_long_prompt_by_a_wide_layer(gated, eight):
    """20001 rows by 14336 columns: more 16-column tiles of rows than threads of a
    grid over 256."""
    from inferkernellab_amd import int4_linear_hip, quantize_rows_int8_hip
    from tests.test_gpu_quantized import _assert_close, _expected, _gen, _sums8, _sums16, _weight

    gen, rows = _gen(3), 20001
    packed, w, mag = _weight(gen, 14336 * (2 if gated else 1), 128, 64, zeros=gated, gated=gated)
    x = torch.randn(rows, 128, generator=gen, device="cuda").to(BF16)
    given = quantize_rows_int8_hip(x, group_size=64) if eight else x
    y = int4_linear_hip(given, packed)
    assert y.shape == (rows, 14336)
    for start in (0, 18700, rows - 65):  # around the last row that the count of tiles once held
        part = slice(start, start + 65)
        if eight:
            codes, scales = given.codes[part], given.scales[part]
            xd = codes.double() * scales.double().repeat_interleave(64, 1)
            sums = _sums8(codes, scales, w, 64)
        else:
            xd = x[part].double()
            sums = _sums16(xd, mag, 64)
        want, bound = _expected(xd, w, sums, None, gated, BF16)
        _assert_close(y[part], want, bound)
