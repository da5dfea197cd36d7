"""The new operators together, as a server runs them: heads normalised and
appended, prompts continued several times on shared pages, pages compacted
between steps, tokens drawn by the sampling kernel."""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_sample import oracle_row

pytestmark = pytest.mark.gpu


def model_of(dtype=torch.bfloat16, *, qk_norm=True, heads=8, kv=2, d=64, layers=3, vocab=515, seed=0):
    from inferkernellab_amd.llama import LlamaConfig, random_llama

    model = random_llama(LlamaConfig(vocab_size=vocab, hidden_size=256, intermediate_size=512, num_hidden_layers=layers,
                                     num_attention_heads=heads, num_key_value_heads=kv, head_dim=d, qk_norm=qk_norm),
                         seed=seed, dtype=dtype)
    gen = torch.Generator().manual_seed(seed + 1)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith("norm.weight"):
                p.copy_((1 + 0.2 * torch.randn(p.shape, generator=gen)).to(p.dtype))
        model.lm_head.weight.mul_(8)  # logits with a spread
    return model


def run(model, prompts, **kw):
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner

    kw.setdefault("max_new_tokens", 9)
    runner = LlamaPagedDecodeRunner(model, prompts, **kw)
    return runner.run(), runner


def prompts_of(lengths, vocab=515, seed=3):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in lengths]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_head_norms_in_one_launch_match_the_modules(dtype, monkeypatch):
    """The fused launch rounds once where the modules round five times: logits
    of the first step agree to a few of the type's steps of their largest."""
    from inferkernellab_amd import ops

    model, prompts = model_of(dtype), prompts_of([5, 33, 17])
    calls = []
    whole = ops.qk_norm_rope_append_kv_hip
    monkeypatch.setattr(ops, "qk_norm_rope_append_kv_hip", lambda *a, **k: calls.append(1) or whole(*a, **k))
    fused, _ = run(model, prompts, use_graph=False)
    assert len(calls) == 3 * (1 + 9)  # a layer's launch for the prefill and each step
    modules, _ = run(model, prompts, append_backend="torch", use_graph=False)
    assert len(calls) == 30
    plain, _ = run(model_of(dtype, qk_norm=False), prompts, use_graph=False)
    a, b = fused.prompt_logits, modules.prompt_logits
    size = b.abs().max()
    tol = {torch.bfloat16: 2.0 ** -5, torch.float16: 2.0 ** -8, torch.float32: 2.0 ** -17}[dtype]
    assert (a - b).abs().max() <= tol * size
    assert (plain.prompt_logits - b).abs().max() > 0.05 * size  # the norms matter


def test_hooked_head_norms_run_as_modules(monkeypatch):
    from inferkernellab_amd import ops

    model, prompts = model_of(), prompts_of([6, 9])
    want, _ = run(model, prompts, use_graph=False)
    seen = []
    for layer in model.model.layers:
        layer.self_attn.q_norm.register_forward_hook(lambda m, i, o: seen.append(o.shape))
    monkeypatch.setattr(ops, "qk_norm_rope_append_kv_hip", None)
    got, _ = run(model, prompts, use_graph=False)
    assert len(seen) == 3 * 10
    assert (got.prompt_logits - want.prompt_logits).abs().max() <= 2.0 ** -5 * want.prompt_logits.abs().max()


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("kv", [None, torch.float8_e4m3fn])
def test_samples_share_the_prompt(use_graph, kv):
    model, prompts = model_of(), prompts_of([5, 33, 16])
    one, _ = run(model, prompts, use_graph=use_graph, kv_cache_dtype=kv)
    three, runner = run(model, prompts, use_graph=use_graph, kv_cache_dtype=kv, num_samples=3)
    assert [r.request_id for r in runner.requests] == list(range(9))
    assert three.cache_released and len(three.generated_tokens) == 9
    whole = 33 // 16 + 16 // 16
    assert three.used_blocks_peak == whole + 3 * (one.used_blocks_peak - whole)
    for i, tokens in enumerate(three.generated_tokens):
        assert torch.equal(three.prompt_logits[i], one.prompt_logits[i // 3])
        assert tokens[:1] == one.generated_tokens[i // 3][:1]
    # three equal rows of one step take equal tokens
    for i in range(0, 9, 3):
        assert three.generated_tokens[i] == three.generated_tokens[i + 1] == three.generated_tokens[i + 2]


@pytest.mark.parametrize("settings", [dict(temperature=0.8), dict(temperature=1.2, top_p=0.8),
                                      dict(temperature=1.0, top_k=7, top_p=0.9), dict(temperature=1.5, min_p=0.1)],
                         ids=str)
def test_drawn_tokens_are_those_of_the_definition(settings):
    """Eager and captured runs draw the definition's token from each step's
    logits and the generators' uniform numbers, and report its log
    probabilities."""
    model, prompts = model_of(), prompts_of([5, 33, 17])
    runs = [run(model, prompts, sampler="hip", num_samples=2, use_graph=g, seed=11, **settings)[0] for g in (False, True)]
    uniform = [torch.rand(9, generator=torch.Generator(device="cuda").manual_seed(11 + i), device="cuda").cpu()
               for i in range(6)]
    assert len({t for r in runs for t in r.generated_tokens}) > 3  # samples differ
    for result in runs:
        for step, logits in enumerate(result.decode_logits):
            for i in range(6):
                want, policy, sampling = oracle_row(logits[i].numpy(), float(uniform[i][step]), np.float32(settings["temperature"]),
                                                    settings.get("top_k", 0), float(np.float32(settings.get("top_p", 1.0))),
                                                    float(np.float32(settings.get("min_p", 0.0))))
                assert result.generated_tokens[i][step] == want
                assert math.isclose(result.token_logprobs[i][step], policy, rel_tol=2.0 ** -24, abs_tol=2.0 ** -28)
                assert math.isclose(result.sampling_logprobs[i][step], sampling, rel_tol=2.0 ** -24, abs_tol=2.0 ** -28)


def test_drawn_tokens_stop_at_eos_and_arguments_are_checked():
    from inferkernellab_amd.llama import LlamaPagedDecodeRunner

    model, prompts = model_of(), prompts_of([7, 12])
    free, _ = run(model, prompts, sampler="hip", temperature=1.0, use_graph=False)
    eos = free.generated_tokens[0][4]
    got, _ = run(model, prompts, sampler="hip", temperature=1.0, eos_token_ids=[eos])
    first = free.generated_tokens[0].index(eos)
    assert got.generated_tokens[0] == free.generated_tokens[0][:first + 1] and got.finish_reasons[0] == "eos"
    greedy, _ = run(model, prompts, sampler="hip", eos_token_ids=[eos])
    plain, _ = run(model, prompts)
    n = len(greedy.generated_tokens[0])
    assert greedy.generated_tokens[0] == plain.generated_tokens[0][:n] and len(greedy.token_logprobs[0]) == n
    for bad in (dict(num_samples=0), dict(sampler="other"), dict(top_k=5), dict(min_p=0.1),
                dict(sampler="hip", top_k=-1), dict(sampler="hip", min_p=2.0)):
        with pytest.raises(ValueError):
            LlamaPagedDecodeRunner(model, prompts, max_new_tokens=2, **bad)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_decode_loop_of_all_of_them(fp8):
    """Two requests prefilled, one forked in the middle of a page, the other
    finished, the pages compacted: what is left attends as a cache that was
    written from the start in one piece."""
    from inferkernellab_amd import (PagedKVCache, paged_decode_attention_hip, qk_norm_rope_append_kv_hip,
                                    sample_tokens_hip)

    heads, kv, d, bs, layers = 8, 2, 64, 16, 2
    gen = torch.Generator().manual_seed(2)
    dtype = torch.bfloat16

    def rows(*shape):
        return torch.randn(*shape, generator=gen).to(dtype).cuda()

    qw, kw = rows(d) * 0.1 + 1, rows(d) * 0.1 + 1
    weight = rows(heads * d, 999) * 0.3
    steps, prompt = 20, 21
    feed = {i: [(rows(1, heads, d), rows(1, kv, d), rows(1, kv, d)) for _ in range(prompt + steps)] for i in (0, 1, 2)}
    angle = torch.rand(prompt + steps, d, generator=gen) * 6
    cos, sin = angle.cos().to(dtype).cuda(), angle.sin().to(dtype).cuda()

    def new_cache(blocks):
        return PagedKVCache(blocks, bs, kv, d, num_layers=layers, device="cuda",
                            dtype=torch.float8_e4m3fn if fp8 else dtype, act_dtype=dtype if fp8 else None)

    def token(cache, table, source, at):
        if at // bs == len(table):
            table += cache.allocator.allocate(1, owner=source)
        slots = cache.slot_mapping(table, at, 1).to(torch.int32)
        outs = []
        for layer in range(layers):
            q, k, v = feed[source][at]
            q = qk_norm_rope_append_kv_hip(q * (layer + 1), k, v, qw, kw, cos[at:at + 1], sin[at:at + 1], cache, slots,
                                           layer, query_out=torch.empty_like(q))
            outs.append(paged_decode_attention_hip(q, cache, [table], [at + 1], layer=layer))
        logits = torch.stack(outs).sum(0).reshape(1, -1).float() @ weight.float()
        u = torch.tensor([(at * 37 % 100) / 100], device="cuda")
        return sample_tokens_hip(logits, u, temperature=0.9, top_k=50, top_p=0.95).item()

    cache = new_cache(12)
    other, parent = cache.allocate_request(1, prompt), cache.allocate_request(0, prompt)
    for at in range(prompt):
        token(cache, other, 1, at)
        token(cache, parent, 0, at)
    child = cache.fork_request(parent, prompt, 2)
    drawn = {0: [], 2: []}
    for at in range(prompt, prompt + steps):
        drawn[0].append(token(cache, parent, 0, at))
        drawn[2].append(token(cache, child, 2, at))
        if at == prompt + 5:
            cache.release_request(other, 1)
            assert cache.compact([parent, child])
    straight = {0: [], 2: []}
    for source in (0, 2):
        whole = new_cache(4)
        table: list[int] = []
        for at in range(prompt + steps):
            got = token(whole, table, source if at >= prompt else 0, at)
            if at >= prompt:
                straight[source].append(got)
    assert drawn == straight and drawn[0] != drawn[2]
    cache.release_request(parent, 0)
    cache.release_request(child, 2)
    assert cache.allocator.num_used_blocks == 0
