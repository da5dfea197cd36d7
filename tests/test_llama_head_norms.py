"""Which norms of query and key heads the Llama runner finds, and at what cost
a layer without them."""

import torch
from torch import nn

from inferkernellab_amd.llama import LlamaConfig, LlamaPagedDecodeRunner, RMSNorm, _Attention

CONFIG = dict(vocab_size=64, hidden_size=32, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,
              num_key_value_heads=1, head_dim=16)


def head_norms(att):
    runner = LlamaPagedDecodeRunner.__new__(LlamaPagedDecodeRunner)
    runner.append_backend, runner.head_dim = "torch", 16
    rows = torch.ones(2, 1, 16)
    return runner._head_norms(att, rows, rows)


def test_a_layer_without_norms_looks_nothing_up_that_is_not_there(monkeypatch):
    """Module attributes that are missing are looked for in Python and raise."""
    att, missing = _Attention(LlamaConfig(**CONFIG)), []
    lookup = nn.Module.__getattr__

    def counted(self, name):
        missing.append(name)
        return lookup(self, name)

    monkeypatch.setattr(nn.Module, "__getattr__", counted)
    assert head_norms(att) is None
    assert missing == []


def test_norms_are_found_however_they_are_held():
    att = _Attention(LlamaConfig(**CONFIG, qk_norm=True))
    assert head_norms(att) == (att.q_norm, att.k_norm, False)
    del att.k_norm
    assert head_norms(att) == (att.q_norm, None, False)
    att = _Attention(LlamaConfig(**CONFIG))
    att.k_norm = lambda x: x  # no module
    assert head_norms(att) == (None, att.k_norm, False)

    class Held(_Attention):
        q_norm = property(lambda self: norm)

    norm = RMSNorm(16, 1e-6)
    assert head_norms(Held(LlamaConfig(**CONFIG))) == (norm, None, False)

    class Wrapped(nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def __getattr__(self, name):
            try:
                return super().__getattr__(name)
            except AttributeError:
                return getattr(self.inner, name)

    att = _Attention(LlamaConfig(**CONFIG, qk_norm=True))
    assert head_norms(Wrapped(att)) == (att.q_norm, att.k_norm, False)
