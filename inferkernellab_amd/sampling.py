"""Drawing the next token of each request from given uniform numbers
(csrc/sample.hip): temperature, top-k, top-p and min-p, with the log
probabilities that the runners report (hf_benchmark.py:578-606, which draws
one request at a time with torch's sort and multinomial and has no top-k or
min-p).

Tokens stand in the order of falling logit, equal ones by index, with the
weight ``exp((logit - max) / temperature)``. Kept are the first ``top_k``; of
those, the tokens whose mass before them is at most ``top_p`` times the mass
of the first ``top_k``; of those, the ones that weigh at least ``min_p`` times
the likeliest. The token drawn is the first whose cumulative mass exceeds the
uniform number's share of the kept mass, so a row's token depends on its
logits, settings and uniform number alone.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .ops import _DTYPES, _INDEX_TYPES, _on_device, _require_backend, _stream


def _setting(value, name: str, rows: int, device: torch.device, fits, wanted: str):
    """(value for all rows, tensor of a value per row or None)."""
    if isinstance(value, torch.Tensor):
        integers = name == "top_k"
        if value.shape != (rows,) or (value.dtype not in _INDEX_TYPES if integers else value.dtype != torch.float32):
            kind = "int32 or int64" if integers else "float32"
            raise ValueError(f"{name} must be a number or a {kind} tensor with one entry per row")
        if value.device != device:
            raise ValueError(f"{name} must be on the logits' device")
        return 0, value
    if not fits(value):
        raise ValueError(f"{name} must be {wanted}")
    return value, None


def _sample_args(logits, uniform, temperature, top_k, top_p, min_p):
    """(argument struct without results and workspace, tensors it points into)."""
    if logits.ndim != 2 or logits.device.type != "cuda":
        raise ValueError("logits must be a GPU (torch 'cuda' device) tensor with shape [B, vocab]")
    if logits.dtype not in _DTYPES:
        raise ValueError("logits dtype must be float16, bfloat16 or float32")
    rows, vocab = logits.shape
    if not 0 < vocab <= _lib.SAMPLE_MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {_lib.SAMPLE_MAX_VOCAB} tokens")
    device = logits.device
    if uniform.shape != (rows,) or uniform.dtype != torch.float32 or uniform.device != device:
        raise ValueError("uniform must be a float32 tensor on the logits' device with one entry per row")
    a = _lib.SampleArgs()
    a.temperature, heat = _setting(temperature, "temperature", rows, device,
                                   lambda v: math.isfinite(v) and v >= 0, "finite and non-negative")
    if a.temperature == 0.0 and heat is None and temperature > 0:
        a.temperature = 2.0 ** -149  # the smallest float32: 0 would state log probabilities at 1
    number, first = _setting(top_k, "top_k", rows, device,
                             lambda v: (isinstance(v, int) or float(v).is_integer()) and v >= 0,
                             "a non-negative whole number")
    a.top_k = min(int(number), vocab)  # any from the vocabulary on keeps every token
    a.top_p, nucleus = _setting(top_p, "top_p", rows, device, lambda v: 0 < v <= 1, "in (0, 1]")
    a.min_p, least = _setting(min_p, "min_p", rows, device, lambda v: 0 <= v <= 1, "in [0, 1]")
    keep = [logits if logits.stride(1) == 1 or vocab == 1 else logits.contiguous()]
    for x in (uniform, heat, first, nucleus, least):
        keep.append(x if x is None or rows <= 1 or x.stride(0) == 1 else x.contiguous())
    logits, uniform, heat, first, nucleus, least = keep
    a.logits, a.logits_stride, a.rows, a.vocab = logits.data_ptr(), logits.stride(0), rows, vocab
    a.dtype = _DTYPES[logits.dtype]
    a.uniform = uniform.data_ptr()
    for name, x in (("temperature_rows", heat), ("top_k_rows", first), ("top_p_rows", nucleus), ("min_p_rows", least)):
        if x is not None:
            setattr(a, name, x.data_ptr())
    if first is not None:
        a.top_k_type = _INDEX_TYPES[first.dtype]
    return a, keep


class PreparedSampler:
    """:func:`sample_tokens_hip` checked once on fixed buffers.

    Binds the logits, the uniform numbers and settings given as tensors, and
    holds the results and the workspace; each call enqueues the draw on the
    current stream and returns the same result tensors. The bound tensors may
    be updated in place between calls. One workspace: calls that may overlap
    need a sampler each.
    """

    def __init__(self, logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, logprobs: bool = False):
        self._lib = _require_backend()
        self._args, self._keep = _sample_args(logits, uniform, temperature, top_k, top_p, min_p)
        given = (logits, uniform, *(v if isinstance(v, torch.Tensor) else None
                                    for v in (temperature, top_k, top_p, min_p)))
        if any(x is not y for x, y in zip(given, self._keep)):
            raise ValueError("tensors of a prepared launch must be contiguous (logits: in their rows)")
        self.device = logits.device
        self._results(logits.shape[0], logprobs)

    def _results(self, rows: int, logprobs: bool) -> None:
        a = self._args
        self.tokens = torch.empty(rows, dtype=torch.int64, device=self.device)
        a.tokens = self.tokens.data_ptr()
        self.policy_logprobs = self.sampling_logprobs = None
        if logprobs:
            self.policy_logprobs = torch.empty(rows, dtype=torch.float32, device=self.device)
            self.sampling_logprobs = torch.empty_like(self.policy_logprobs)
            a.policy_logprobs = self.policy_logprobs.data_ptr()
            a.sampling_logprobs = self.sampling_logprobs.data_ptr()
        size = self._lib.ikl_sample_workspace_size(ctypes.byref(a))
        _lib.check(min(size, 0), "sample")
        self.workspace = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        a.workspace, a.workspace_bytes = self.workspace.data_ptr() if size else None, size
        self._out = (self.tokens, self.policy_logprobs, self.sampling_logprobs) if logprobs else self.tokens

    def __call__(self):
        with _on_device(self.device):
            status = self._lib.ikl_sample_tokens(ctypes.byref(self._args), _stream(self.device))
        _lib.check(status, "sample")
        return self._out


def sample_tokens_hip(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                      logprobs: bool = False):
    """Draw one token per row of ``logits`` ``[B, vocab]`` (fp16, bf16, fp32).

    ``uniform`` ``[B]`` float32 in [0, 1) decides the draw. ``temperature``,
    ``top_k``, ``top_p`` and ``min_p`` are numbers, or tensors with one entry
    per row (float32; ``top_k`` int32 / int64), whose values are not looked at
    on the host: one outside its range acts as the nearest inside. Temperature
    0 takes the likeliest token, ``top_k=0``, ``top_p=1`` and ``min_p=0`` keep
    every token. NaN logits count as -inf; a row with nothing above -inf gets
    token -1 and log probabilities -inf.

    Returns the tokens ``[B]`` int64; with ``logprobs`` also the float32 log
    probability of each under all tokens at the temperature (1 where that is
    0) and among the tokens kept.
    """
    call = PreparedSampler.__new__(PreparedSampler)
    call._lib = _require_backend()
    call._args, call._keep = _sample_args(logits, uniform, temperature, top_k, top_p, min_p)
    call.device = logits.device
    call._results(logits.shape[0], logprobs)
    return call()
