"""The scales of K rows that the normalised append quantises: the smallest power
of two that keeps the row within E4M3's range, 1 for a row of zeros, and nothing
changed outside the slots.

Tolerance: the fp32 row differs from the formula by at most F32_STEPS of
|y1 cos| + |y2 sin| (tests/test_gpu_norm_rope.py), so its largest magnitude by
F32_STEPS of the largest of these; only within that of a border may the scale be
the border's other side. A value is then off by half a step of E4M3 (2^-4 of it,
or half the smallest step, 2^-10 of the scale) and the fp32 row's own error."""

import pytest
import torch

from tests.test_gpu_norm_rope import F32_STEPS, formula, make


def check_rows(values, scale, ref, mag):
    """Values and scales [T, H] of rows whose float64 formula gives `ref` [T, H, D]."""
    part, power = torch.frexp(scale)
    assert (part == 0.5).all(), "a scale is no power of two"
    most, off = ref.abs().amax(-1), F32_STEPS * mag.amax(-1)
    zero = most == 0
    assert (scale[zero] == 1).all()
    s, most, off = scale.double()[~zero], most[~zero], off[~zero]
    assert (448 * s >= most - off).all(), "a row leaves E4M3's range"
    assert ((224 * s <= most + off) | (s == 2.0 ** -126)).all(), "a scale is larger than the row needs"
    err = (values.double() - ref).abs()
    assert (err <= ref.abs() * 2.0 ** -4 + 2.0 ** -10 * scale.double()[..., None] + 2 * F32_STEPS * mag).all()


def rows_of(seed=0, tokens=40, heads=3, d=64):
    gen = torch.Generator().manual_seed(seed)
    ref = torch.randn(tokens, heads, d, generator=gen, dtype=torch.float64)
    ref *= 2.0 ** torch.randint(-30, 20, (tokens, heads, 1), generator=gen)
    ref[3, 1] = 0
    return ref


def quantised(ref, scale):
    codes = (ref.float() / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.float() * scale[..., None]


def test_the_check_finds_planted_mistakes():
    from inferkernellab_amd.cache import quantize_rows_e4m3

    ref = rows_of()
    scale = quantize_rows_e4m3(ref.float())[1]
    check_rows(quantised(ref, scale), scale, ref, ref.abs())
    for wrong in (torch.ones_like(scale), scale * 2, scale / 2, scale * 1.5,
                  torch.where(scale == scale.max(), scale / 2, scale)):
        with pytest.raises(AssertionError):
            check_rows(quantised(ref, wrong), wrong, ref, ref.abs())
    values = quantised(ref, scale)
    values[7, 2, 5] *= 1.25
    with pytest.raises(AssertionError):
        check_rows(values, scale, ref, ref.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv,d,head_major", [(1, 32, 8, 128, True), (33, 4, 2, 64, False),
                                                          (517, 16, 4, 96, True), (9, 2, 1, 512, False),
                                                          (300, 8, 8, 32, True)])
def test_scales_of_the_appended_rows(dtype, tokens, heads, kv, d, head_major):
    from inferkernellab_amd import qk_norm_rope_append_kv_hip
    from inferkernellab_amd.cache import quantize_rows_e4m3

    case = make(dtype, tokens, heads, kv, d, fp8=True, head_major=head_major)
    cache, slots = case["cache"], case["slots"].long()
    case["key"][tokens // 2, 0] = 0
    # weights over the type's range give rows of many sizes
    case["k_weight"] = case["k_weight"].repeat(kv, 1) * (2.0 ** torch.arange(kv, device="cuda") / 16)[:, None].to(dtype)
    gen = torch.Generator(device="cuda").manual_seed(7)
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.rand(t.shape, generator=gen, device="cuda"))
    before = [t.clone() for t in (cache.k_scale, cache.v_scale, cache.k.view(torch.uint8), cache.v.view(torch.uint8))]
    out = torch.empty_like(case["query"])
    qk_norm_rope_append_kv_hip(case["query"], case["key"], case["value"], case["q_weight"], case["k_weight"], case["cos"],
                               case["sin"], cache, case["slots"], 1, eps=1e-6, query_out=out)
    block, place = slots // cache.layout.block_size, slots % cache.layout.block_size
    ref, mag = formula(case["key"], case["k_weight"], case["cos"], case["sin"], 1e-6)
    scale = cache.k_scale[1, block, :, place]
    check_rows(cache.k.float()[1, block, place] * scale[..., None], scale, ref, mag)
    codes, vs = quantize_rows_e4m3(case["value"])
    assert torch.equal(cache.v_scale[1, block, :, place], vs)
    assert torch.equal(cache.v.view(torch.uint8)[1, block, place], codes.view(torch.uint8))
    for t, old in zip((cache.k_scale, cache.v_scale), before[:2]):
        same = t == old
        same[1, block, :, place] = True
        assert same.all(), "a scale outside the slots changed"
    for t, old in zip((cache.k, cache.v), before[2:]):
        same = t.view(torch.uint8) == old
        same[1, block, place] = True
        assert same.all(), "a row outside the slots changed"
