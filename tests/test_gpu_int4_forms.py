"""Products over 4-bit weights by every form of a launch, each type of rows and
of results; a gated MLP by its values; the Llama runner over fp16, and its
decoded logits step by step."""

import pytest
import torch

from tests.int4_forms import FORMS, cols_of, plan
from tests.test_gpu_llama_int4 import _model, _plain_int8, _prompts
from tests.test_gpu_quantized import BF16, FP16, FP32, _assert_close, _expected, _gen, _sums8, _sums16, _weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight,dtype", [(False, BF16), (False, FP16), (True, BF16), (True, FP16), (True, FP32)],
                         ids=["bf16", "fp16", "8 bits to bf16", "8 bits to fp16", "8 bits to fp32"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_every_form_of_a_launch(eight, dtype, group, zeros):
    """Contractions that end inside a step (groups of 32 and 64), with and
    without a residual, of which half the products' rows are in wide buffers."""
    from inferkernellab_amd import _lib, int4_linear_hip, quantize_rows_int8_hip

    code = {BF16: _lib.IKL_BF16, FP16: _lib.IKL_F16, FP32: _lib.IKL_F32}[dtype]
    for n, (of_eight, gated, form, parts, rows, outs, steps) in enumerate(FORMS):
        if of_eight != eight:
            continue
        cols = cols_of(steps, group)
        taken, split = plan(eight, gated, rows, outs, cols, group, code)
        assert (taken, split > 1) == (form, parts)
        gen = _gen(n)
        packed, w, mag = _weight(gen, outs * (2 if gated else 1), cols, group, zeros=zeros, gated=gated)
        x = torch.randn(rows, cols, generator=gen, device="cuda").to(dtype)
        res = None
        if not gated and (n + zeros) % 2:
            res = torch.randn(rows, outs + 8, generator=gen, device="cuda").to(dtype)[:, 3:outs + 3]
        if eight:
            x = quantize_rows_int8_hip(x, group_size=group)
            xd = (x.codes.double().view(rows, -1, group) * x.scales.double()[..., None]).view(rows, cols)
            sums = _sums8(x.codes, x.scales, w, group)
        else:
            xd = x.double()
            sums = _sums16(xd, mag, group)
        want, bound = _expected(xd, w, sums, res, gated, dtype)
        out = torch.full((rows, outs + 16), 5.0, dtype=dtype, device="cuda")
        y = int4_linear_hip(x, packed, residual=res, out=out[:, 8:outs + 8])
        _assert_close(y, want, bound)
        assert bool((out[:, :8] == 5).all()) and bool((out[:, outs + 8:] == 5).all())
        assert torch.equal(int4_linear_hip(x, packed, residual=res), y)


@pytest.mark.parametrize("rows", [1, 29, 150])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("eight", [False, True])
def test_a_gated_mlp_by_its_values(rows, dtype, eight):
    """norm -> gated product -> 8 bits -> down + residual."""
    from inferkernellab_amd import add_rms_norm_int8_hip, int4_linear_hip, quantize_rows_int8_hip

    gen = _gen(rows)
    hidden, inner, group = 512, 704, 64
    x, delta = torch.randn(2, rows, hidden, generator=gen, device="cuda").to(dtype)
    norm = (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).to(dtype)
    gate_up, wgu, mgu = _weight(gen, 2 * inner, hidden, group, zeros=True, gated=True)
    down, wd, md = _weight(gen, hidden, inner, group, zeros=False)
    total, rows8 = add_rms_norm_int8_hip(x, delta, norm, group_size=group)

    def stands(r):
        return (r.codes.double().view(rows, -1, group) * r.scales.double()[..., None]).view(rows, -1)

    if eight:
        act = int4_linear_hip(rows8, gate_up)
        _assert_close(act, *_expected(stands(rows8), wgu, _sums8(rows8.codes, rows8.scales, wgu, group), None, True,
                                      dtype))
        given = quantize_rows_int8_hip(act, group_size=group)
        a, sums = stands(given), _sums8(given.codes, given.scales, wd, group)
    else:
        plain = rows8.dequantize()
        given = act = int4_linear_hip(plain, gate_up)
        _assert_close(act, *_expected(plain.double(), wgu, _sums16(plain.double(), mgu, group), None, True, dtype))
        a, sums = act.double(), _sums16(act.double(), md, group)
    _assert_close(int4_linear_hip(given, down, residual=total), *_expected(a, wd, sums, total, False, dtype))


def test_fp16_run_matches_the_oracle_of_the_same_weights():
    """As the bf16 run, whose tolerance counts 8 roundings to bf16: so many to
    fp16, whose steps are an eighth."""
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner, quantize_llama_int4
    from tests.test_gpu_runners import _check_llama

    cfg, model = _model(FP16)
    prompts = _prompts(70, 33, 129, 5)
    w = quantize_llama_int4(model, group_size=64)
    result = LlamaPagedDecodeRunner(model, prompts, max_new_tokens=6, max_num_batched_tokens=128, int4_weights=w).run()
    assert result.cache_released and result.prefill_batch_count > 1
    _check_llama(cfg, model, result, prompts, tol=3e-2 / 8, margin_check=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decoded_logits_match_the_plain_operators_step_by_step(monkeypatch, dtype):
    """Rows in 8 bits: a request's logits of each step that the same tokens lead
    to, the first in any case. (The plain product rounds to bf16 whatever the
    run's type.)"""
    from inferkernellab_amd import llama
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner, quantize_llama_int4

    _, model = _model(dtype)
    w = quantize_llama_int4(model, group_size=64, symmetric=False)
    run = dict(max_new_tokens=6, max_num_batched_tokens=48, int4_weights=w, int8_rows=True, use_graph=False)
    got = LlamaPagedDecodeRunner(model, _prompts(70, 33, 5), **run).run()
    _plain_int8(monkeypatch)
    plain = llama.int4_linear_hip
    monkeypatch.setattr(llama, "int4_linear_hip", lambda *a, **kw: plain(*a, **kw).to(dtype))
    ref = LlamaPagedDecodeRunner(model, _prompts(70, 33, 5), **run).run()
    scale = float(ref.prompt_logits.abs().max())
    assert float((got.prompt_logits - ref.prompt_logits).abs().max()) <= 3e-2 * scale
    compared = 0
    for r in range(3):
        for step, (a, b) in enumerate(zip(got.decode_logits, ref.decode_logits)):
            if got.generated_tokens[r][:step] != ref.generated_tokens[r][:step]:
                break
            assert float((a[r] - b[r]).abs().max()) <= 6e-2 * scale, (r, step)
            compared += 1
    assert compared >= 3
