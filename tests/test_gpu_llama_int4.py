"""The Llama runner over 4-bit weights. The models' linear weights lie on the
4-bit grid (whole numbers of -7 to 7 times a power of two, a 7 in every group),
so that rounding them to 4 bits changes nothing and the runs can be held to the
same model's oracle."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(dtype=torch.bfloat16, seed=5, **kw):
    from inferkernellab_amd.llama import LlamaConfig, random_llama

    cfg = LlamaConfig(**{**dict(vocab_size=256, hidden_size=512, intermediate_size=704, num_hidden_layers=2,
                                num_attention_heads=8, num_key_value_heads=2), **kw})
    model = random_llama(cfg, seed=seed, device="cuda", dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for layer in model.model.layers:
        for lin in (m for m in layer.modules() if isinstance(m, torch.nn.Linear)):
            c = torch.randint(-7, 8, lin.weight.shape, generator=gen, device="cuda")
            c[:, ::32] = 7
            with torch.no_grad():
                lin.weight.copy_(c * 2.0**-8)
    return cfg, model


def _prompts(*lengths):
    gen = torch.Generator().manual_seed(1)
    return [torch.randint(0, 256, (n,), generator=gen).tolist() for n in lengths]


@pytest.mark.parametrize("group", [32, 64])
def test_weights_on_the_grid_are_kept(group):
    from inferkernellab_amd.llama import quantize_llama_int4

    _, model = _model()
    w = quantize_llama_int4(model, group_size=group)
    for layer, q in zip(model.model.layers, w.layers):
        a, m = layer.self_attn, layer.mlp
        for packed, parts in ((q.qkv, (a.q_proj, a.k_proj, a.v_proj)), (q.o, (a.o_proj,)),
                              (q.gate_up, (m.gate_proj, m.up_proj)), (q.down, (m.down_proj,))):
            assert torch.equal(packed.dequantize(), torch.cat([p.weight.float() for p in parts]))


def test_bf16_run_matches_the_oracle_of_the_same_weights():
    """Against the CPU oracle in bf16, as the run over 16-bit weights."""
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner, quantize_llama_int4
    from tests.test_gpu_runners import _check_llama

    cfg, model = _model()
    prompts = _prompts(70, 33, 129, 5)
    w = quantize_llama_int4(model, group_size=64)
    result = LlamaPagedDecodeRunner(model, prompts, max_new_tokens=6, max_num_batched_tokens=128, int4_weights=w).run()
    assert result.cache_released and result.prefill_batch_count > 1
    _check_llama(cfg, model, result, prompts, tol=3e-2, margin_check=True)


def _plain_int8(monkeypatch):
    """The runner's quantised operators in torch, 64 bits, rounded once."""
    from inferkernellab_amd import llama

    def grid(v, group):
        g = v.reshape(*v.shape[:-1], -1, group)
        step = g.abs().amax(-1, keepdim=True).clamp(min=2.0**-100) / 127
        return ((g / step).round() * step).view(v.shape)

    def rows(x, group_size):
        return grid(x.double(), group_size)

    def norm(x, delta, weight, eps, group_size):
        total = x if delta is None else x + delta
        t = total.double()
        return total, grid(t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * weight.double(), group_size)

    def linear(x, weight, residual=None):
        y = x.double() @ weight.dequantize(torch.float64).t().contiguous()
        if weight.gated:
            gate, up = y.chunk(2, -1)
            y = gate * torch.sigmoid(gate) * up
        return (y if residual is None else y + residual.double()).to(torch.bfloat16)

    monkeypatch.setattr(llama, "quantize_rows_int8_hip", rows)
    monkeypatch.setattr(llama, "add_rms_norm_int8_hip", norm)
    monkeypatch.setattr(llama, "int4_linear_hip", linear)


@pytest.mark.parametrize("kw", [dict(), dict(kv_cache_dtype=torch.float8_e4m3fn), dict(append_backend="torch"),
                                dict(qk_norm=True)], ids=str)
def test_rows_in_8_bits_match_the_plain_operators(monkeypatch, kw):
    """Chunked ragged prompts and decoded tokens; the bf16 logits of the two
    part where a rounding falls the other way."""
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner, quantize_llama_int4

    kw = dict(kw)
    _, model = _model(qk_norm=kw.pop("qk_norm", False))
    w = quantize_llama_int4(model, group_size=64, symmetric=False)
    run = dict(max_new_tokens=4, max_num_batched_tokens=48, int4_weights=w, int8_rows=True, use_graph=False, **kw)
    got = LlamaPagedDecodeRunner(model, _prompts(70, 33, 5), **run).run()
    _plain_int8(monkeypatch)
    ref = LlamaPagedDecodeRunner(model, _prompts(70, 33, 5), **run).run()
    scale = float(ref.prompt_logits.abs().max())
    assert float((got.prompt_logits - ref.prompt_logits).abs().max()) <= 3e-2 * scale
    if got.generated_tokens == ref.generated_tokens:
        for a, b in zip(got.decode_logits, ref.decode_logits):
            assert float((a - b).abs().max()) <= 6e-2 * scale


@pytest.mark.parametrize("int8_rows", [False, True])
def test_captured_steps_give_the_eager_tokens(int8_rows):
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner, quantize_llama_int4

    _, model = _model()
    w = quantize_llama_int4(model, group_size=32)
    kw = dict(max_new_tokens=7, int4_weights=w, int8_rows=int8_rows, num_samples=2, temperature=0.9, sampler="hip")
    captured = LlamaPagedDecodeRunner(model, _prompts(19, 40, 3), **kw).run()
    eager = LlamaPagedDecodeRunner(model, _prompts(19, 40, 3), use_graph=False, **kw).run()
    assert captured.generated_tokens == eager.generated_tokens
    for a, b in zip(captured.decode_logits, eager.decode_logits):
        assert torch.equal(a, b)


def test_a_norm_that_is_no_plain_one_runs_as_its_module():
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner, RMSNorm, quantize_llama_int4

    class Norm(RMSNorm):
        def forward(self, x):
            self.calls = getattr(self, "calls", 0) + 1
            return super().forward(x)

    _, model = _model()
    w = quantize_llama_int4(model, group_size=64)
    kw = dict(max_new_tokens=3, int4_weights=w, int8_rows=True)
    plain = LlamaPagedDecodeRunner(model, _prompts(9, 30), **kw).run()
    for layer in model.model.layers:
        layer.input_layernorm = Norm(512, 1e-6).to("cuda", torch.bfloat16).requires_grad_(False)
    own = LlamaPagedDecodeRunner(model, _prompts(9, 30), **kw).run()
    assert all(layer.input_layernorm.calls > 0 for layer in model.model.layers)
    scale = float(plain.prompt_logits.abs().max())
    assert float((plain.prompt_logits - own.prompt_logits).abs().max()) <= 3e-2 * scale
