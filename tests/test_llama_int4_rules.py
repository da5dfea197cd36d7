"""What 4-bit weights of a Llama model refuse: modules that the kernels would
not restate, and weights of another model."""

import pytest
import torch
from torch import nn

from inferkernellab_amd.llama import LlamaConfig, LlamaPagedDecodeRunner, quantize_llama_int4, random_llama


def _model(dtype=torch.bfloat16, **kw):
    cfg = LlamaConfig(**{**dict(vocab_size=32, hidden_size=64, intermediate_size=128, num_hidden_layers=2,
                                num_attention_heads=2, num_key_value_heads=1), **kw})
    return random_llama(cfg, seed=0, device="cpu", dtype=dtype)


def _check(model, weights):
    runner = LlamaPagedDecodeRunner.__new__(LlamaPagedDecodeRunner)
    runner.model, runner.dtype, runner.device = model, next(model.parameters()).dtype, torch.device("cpu")
    runner._check_int4(weights)


def test_a_models_own_weights_fit():
    model = _model()
    w = quantize_llama_int4(model, group_size=32)
    _check(model, w)
    assert w.layers[0].qkv.out_features == 64 + 32 + 32 and w.layers[1].gate_up.gated
    att = model.model.layers[0].self_attn
    stacked = torch.cat([m.weight for m in (att.q_proj, att.k_proj, att.v_proj)]).float()
    step = w.layers[0].qkv.dequantize() - stacked
    assert float(step.abs().max()) <= float(stacked.abs().max()) / 7 * 0.5 * (1 + 2.0**-4)


def _bias(layer):
    layer.mlp.down_proj = nn.Linear(128, 64, dtype=torch.bfloat16)


def _hook(layer):
    layer.self_attn.k_proj.register_forward_hook(lambda *a: None)


def _subclass(layer):
    class Other(nn.Linear):
        pass

    layer.self_attn.o_proj = Other(64, 64, bias=False, dtype=torch.bfloat16)


def _activation(layer):
    layer.mlp.act_fn = nn.GELU()


@pytest.mark.parametrize("change", [_bias, _hook, _subclass, _activation])
def test_modules_that_are_no_plain_linears(change):
    model = _model()
    w = quantize_llama_int4(model, group_size=32)
    change(model.model.layers[1])
    with pytest.raises(ValueError, match="4-bit weights"):
        quantize_llama_int4(model, group_size=32)
    with pytest.raises(ValueError, match="4-bit weights"):
        _check(model, w)


def test_weights_of_another_model():
    w = quantize_llama_int4(_model(), group_size=32)
    for other in (_model(num_hidden_layers=1), _model(hidden_size=128), _model(intermediate_size=96),
                  _model(num_key_value_heads=2), _model(dtype=torch.float32)):
        with pytest.raises(ValueError, match="int4_weights"):
            _check(other, w)
    with pytest.raises(ValueError, match="whole groups"):
        quantize_llama_int4(_model(), group_size=128)


def test_rows_in_8_bits_need_4_bit_weights():
    with pytest.raises(ValueError, match="int8_rows needs int4_weights"):
        LlamaPagedDecodeRunner(_model(), [[1]], max_new_tokens=1, int8_rows=True)
