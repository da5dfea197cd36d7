"""Cases of the decode step's sampling, normalised rotary append and page copies.

A case is a dict of plain values; ``kind`` names the operator:

* ``sample``: one token per row of logits with temperature, top-k, top-p and
  min-p from given uniform numbers (``PreparedSampler``), with the log
  probabilities of the drawn tokens;
* ``norm_rope``: RMSNorm of each query and key head, rotate-half RoPE and the
  append of k and v to the paged cache (``PreparedQKNormRopeAppend``);
* ``copy``: pages copied to other pages over all layers of the cache, as a
  fork or a compaction does (``copy_blocks_hip``).

Where ``own`` is false the operators run in their plain form: elementary torch
operations, in 64 bits for the sampling (whole tokens hang on sums and borders)
and in 32 bits for the norm and the rotation.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"
EPS = 1e-6


def listed():
    return [
        # The smallest draw: one request answered in a chat, a 32000-token
        # vocabulary, nucleus sampling.
        _sample("sample_b1_topp", 1, 32000, "bf16", 0.7, 0, 0.9, 0.0),
        # A small batch with the usual top-k and top-p together.
        _sample("sample_b16_topk_topp", 16, 32000, "bf16", 0.8, 50, 0.95, 0.0),
        # Requests of different settings in one batch, an odd vocabulary.
        _sample("sample_b61_mixed", 61, 50257, "fp16", 1.0, 0, 1.0, 0.0, mixed=True),
        # Plain temperature sampling over a large vocabulary, banned tokens
        # at -inf.
        _sample("sample_b32_temperature", 32, 131072, "bf16", 1.0, 0, 1.0, 0.0, banned=0.02),
        # The largest: a full batch, fp32 logits, a wide nucleus.
        _sample("sample_b256_topp", 256, 131072, "fp32", 1.2, 0, 0.95, 0.02),
        # One token of one request: latency.
        _norm_rope("norm_rope_t1", 1, 32, 8, 128, "bf16"),
        # A decode batch into the FP8 cache.
        _norm_rope("norm_rope_t32_fp8", 32, 32, 8, 128, "bf16", cache="fp8"),
        # An odd chunk of a small model.
        _norm_rope("norm_rope_t517", 517, 16, 4, 64, "fp16"),
        # A batched prefill's rows.
        _norm_rope("norm_rope_t8192", 8192, 32, 8, 128, "bf16"),
        # A request forked in the middle of a page, an 8-layer model.
        _copy("copy_fork_1", 1, 8, 64, 16, 4, 128, "bf16"),
        # A batch forked for parallel samples, a 32-layer model.
        _copy("copy_fork_32", 32, 32, 256, 16, 8, 128, "bf16"),
        # A compaction that moves a third of a large cache.
        _copy("copy_compact_512", 512, 16, 1536, 16, 8, 128, "bf16"),
    ]


def draw(rng):
    kind = rng.choice(("sample", "sample", "norm_rope", "copy"))
    if kind == "sample":
        vocab = rng.choice((_spread(rng, 255, 131072), 32000, 50257, 128001))
        rows = min(_spread(rng, 1, 256), max(1, 256 * 131072 // vocab))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        return _sample(None, rows, vocab, dtype, rng.choice((0.0, 0.3, 0.7, 1.0, 1.3)),
                       rng.choice((0, 0, 1, 20, 50, 300)), rng.choice((1.0, 0.5, 0.8, 0.9, 0.95, 0.99)),
                       rng.choice((0.0, 0.0, 0.02, 0.1)), mixed=rng.random() < 0.3,
                       banned=rng.choice((0.0, 0.0, 0.02, 0.5)))
    if kind == "norm_rope":
        heads, kv_heads = rng.choice(((32, 8), (16, 4), (4, 2), (32, 32), (8, 1)))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        cache = "fp8" if dtype != "fp32" and rng.random() < 0.25 else "same"
        most = 8192 if dtype != "fp32" else 2048
        return _norm_rope(None, _spread(rng, 1, most), heads, kv_heads, rng.choice((32, 64, 96, 128)), dtype,
                          cache=cache, block=rng.choice((16, 32)))
    layers, blocks = rng.choice((1, 8, 16, 32)), _spread(rng, 64, 768)
    return _copy(None, _spread(rng, 1, blocks // 3), layers, blocks, rng.choice((8, 16, 32)),
                 rng.choice((1, 2, 4)), rng.choice((64, 128)), rng.choice(("bf16", "fp16", "fp32")))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"sample": _prepare_sample, "norm_rope": _prepare_norm_rope, "copy": _prepare_copy}[case["kind"]](case, gen)
    if own:
        _bind(case, state)
    return {"case": case, **state}


def run(state):
    if own:
        return _own(state)
    return {"sample": _plain_sample, "norm_rope": _plain_norm_rope, "copy": _plain_copy}[state["case"]["kind"]](state)


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        # a row's logits once, its settings and its three results; a subtraction,
        # a division, an exponential and a sum for each logit
        return {"bytes": n * _size(case) + case["rows"] * (20 + 16), "flops": 4.0 * n}
    if case["kind"] == "norm_rope":
        t, h, hkv, d, eb = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], _size(case)
        read = t * ((h + 2 * hkv + 2) * d * eb + 8) + 2 * d * eb
        kv = t * 2 * hkv * (d + 4 if case["cache"] == "fp8" else d * eb)
        return {"bytes": read + t * h * d * eb + kv, "flops": t * (h + hkv) * d * 7.0}
    page = case["block"] * case["kv_heads"] * case["head_dim"] * _size(case)
    return {"bytes": 2.0 * 2 * case["pairs"] * case["layers"] * page + 8 * case["pairs"], "flops": 0}


def exact(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "sample":
        return _exact_sample(_prepare_sample(case, gen))
    if case["kind"] == "norm_rope":
        return _exact_norm_rope(case, _prepare_norm_rope(case, gen))
    return None  # a copy computes no numbers


# ------------------------------------------------------------------ the cases
def _size(case):
    return DTYPES[case["dtype"]].itemsize


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _sample(name, rows, vocab, dtype, temperature, top_k, top_p, min_p, *, mixed=False, banned=0.0):
    """`mixed`: the rows' settings differ, drawn with the inputs; `banned`: the share of logits at -inf."""
    return _named(name, {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature,
                         "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "banned": banned})


def _norm_rope(name, tokens, heads, kv_heads, head_dim, dtype, *, cache="same", block=16):
    return _named(name, {"kind": "norm_rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
                         "head_dim": head_dim, "dtype": dtype, "cache": cache, "block": block})


def _copy(name, pairs, layers, blocks, block, kv_heads, head_dim, dtype):
    return _named(name, {"kind": "copy", "pairs": pairs, "layers": layers, "blocks": blocks, "block": block,
                         "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype})


# ------------------------------------------------------------------- sampling
def _prepare_sample(case, gen):
    b, v = case["rows"], case["vocab"]

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    # a normal bulk and a few likely tokens, as a language model's head gives
    logits = torch.randn(b, v, generator=gen, device=DEVICE) * 2.0
    head = torch.randint(0, v, (b, 40), generator=gen, device=DEVICE)
    logits.scatter_add_(1, head, uniform(b, 40) * 11.0)
    if case["banned"]:
        logits.masked_fill_(uniform(b, v) < case["banned"], -math.inf)
        logits[:, 0] = 1.0  # one token at least may be drawn
    ones = torch.ones(b, device=DEVICE)
    state = {"logits": logits.to(DTYPES[case["dtype"]]), "uniform": uniform(b), "temperature": ones * case["temperature"],
             "top_k": torch.full((b,), case["top_k"], dtype=torch.int32, device=DEVICE), "top_p": ones * case["top_p"],
             "min_p": ones * case["min_p"]}
    if case["mixed"]:
        def pick(values, dtype=torch.float32):
            at = torch.randint(0, len(values), (b,), generator=gen, device=DEVICE)
            return torch.tensor(values, dtype=dtype, device=DEVICE)[at]

        state |= {"temperature": pick((0.0, 0.6, 0.8, 1.0, 1.5)), "top_k": pick((0, 1, 40, 200), torch.int32),
                  "top_p": pick((1.0, 0.9, 0.95)), "min_p": pick((0.0, 0.05))}
    return state


def _plain_sample(state):
    """Order the logits, weigh them, strike out what the settings leave out and
    take the first token whose cumulative mass passes the uniform's share."""
    x = state["logits"].double()
    vocab = x.shape[1]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = state["temperature"] == 0
    heat = torch.where(greedy, 1.0, state["temperature"].double())[:, None]
    top = x[:, :1]
    weight = torch.exp((x - top) / heat)
    total = weight.sum(1, keepdim=True)
    top_k = state["top_k"][:, None]
    rank = torch.arange(vocab, device=x.device)[None]
    kept = weight * ((rank < top_k) | (top_k == 0))
    mass = kept.cumsum(1)
    kept = kept * (mass - kept <= state["top_p"].double()[:, None] * mass[:, -1:])
    kept = kept * (weight >= state["min_p"].double()[:, None])
    mass = kept.cumsum(1)
    left = mass[:, -1:]
    target = torch.where(greedy, 0.0, state["uniform"].double())[:, None] * left
    place = (mass <= target).sum(1, keepdim=True)
    place = torch.minimum(place, (kept > 0).sum(1, keepdim=True) - 1)
    share = (x.gather(1, place) - top) / heat
    return {"tokens": order.gather(1, place)[:, 0], "policy": (share - total.log())[:, 0].float(),
            "sampling": (share - left.log())[:, 0].float()}


def _exact_sample(state):
    """Row by row: the log probabilities of the tokens, from the definition. The
    sorted order is made of (logit, index) pairs."""
    tokens, policy, sampling = [], [], []
    for b in range(state["logits"].shape[0]):
        x = state["logits"][b].to(torch.float64)
        t, k = float(state["temperature"][b]), int(state["top_k"][b])
        p, q, u = float(state["top_p"][b]), float(state["min_p"][b]), float(state["uniform"][b])
        alive = torch.nonzero(x > -math.inf)[:, 0]
        by_index = alive[torch.argsort(x[alive].neg(), stable=True)]
        logw = (x[by_index] - x[by_index[0]]) / (t if t > 0 else 1.0)
        w = logw.exp()
        n = min(k, w.numel()) if k > 0 else w.numel()
        before = torch.cat((w.new_zeros(1), w[:n].cumsum(0)))
        n = min(n, int((before[:n] <= p * before[n]).sum()), max(1, int((w >= q).sum())))
        aim = (u if t > 0 else 0.0) * before[n]
        at = min(n - 1, int(torch.searchsorted(before[1:n + 1].contiguous(), aim.reshape(1), right=True)))
        tokens.append(by_index[at])
        policy.append(logw[at] - torch.logsumexp(logw, 0))
        sampling.append(logw[at] - torch.logsumexp(logw[:n], 0))
    return {"tokens": torch.stack(tokens), "policy": torch.stack(policy), "sampling": torch.stack(sampling)}


# -------------------------------------------------- norm, rotation and append
def _prepare_norm_rope(case, gen):
    t, h, hkv, d, bs = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "block"))
    dtype = DTYPES[case["dtype"]]
    blocks = -(-t // bs) + 3

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)

    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEVICE) / d)
    position = torch.randint(0, 8192, (t, 1), generator=gen, device=DEVICE).double()
    angle = torch.cat((position * inv, position * inv), 1)
    shape = (1, blocks, bs, hkv, d)
    state = {"query": normal(t, h, d) * 2, "key": normal(t, hkv, d) * 2, "value": normal(t, hkv, d),
             "q_weight": normal(d) * 0.1 + 1, "k_weight": normal(d) * 0.1 + 1, "cos": angle.cos().to(dtype),
             "sin": angle.sin().to(dtype), "query_out": torch.empty(t, h, d, dtype=dtype, device=DEVICE),
             "slots": torch.randperm(blocks * bs, generator=gen, device=DEVICE)[:t].to(torch.int32)}
    if case["cache"] == "fp8":  # a block's rows of one head together
        store = (1, blocks, hkv, bs, d)
        state["k"] = torch.zeros(store, dtype=torch.float8_e4m3fn, device=DEVICE).transpose(2, 3)
        state["v"] = torch.zeros(store, dtype=torch.float8_e4m3fn, device=DEVICE).transpose(2, 3)
        state["k_scale"] = torch.ones(1, blocks, hkv, bs, device=DEVICE)
        state["v_scale"] = torch.ones(1, blocks, hkv, bs, device=DEVICE)
    else:
        state["k"] = torch.zeros(shape, dtype=dtype, device=DEVICE)
        state["v"] = torch.zeros(shape, dtype=dtype, device=DEVICE)
    return state


def _plain_norm_rope(state):
    cos, sin = state["cos"].float()[:, None], state["sin"].float()[:, None]

    def turned(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        half = x.shape[-1] // 2
        return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin

    query = turned(state["query"], state["q_weight"])
    key = turned(state["key"], state["k_weight"])
    state["query_out"].copy_(query)
    size = state["k"].shape[2]
    slots = state["slots"].long()
    block, place = slots // size, slots % size
    if "k_scale" not in state:
        state["k"][0, block, place] = key.to(state["k"].dtype)
        state["v"][0, block, place] = state["value"]
        return state["query_out"], state["k"], state["v"]
    for name, rows in (("k", key), ("v", state["value"].float())):
        step = _row_scale(rows)
        state[name][0, block, place] = (rows / step[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        state[name + "_scale"][0, block, :, place] = step
    return state["query_out"], _values(state, "k"), _values(state, "v")


def _row_scale(rows):
    """The power of two at or above a row's largest magnitude over 448; 1 for a row of zeros."""
    most = rows.abs().amax(-1)
    part, power = torch.frexp(most / 448.0)
    power = torch.where(part == 0.5, power - 1, power).clamp(min=-126)
    return torch.where(most > 0, torch.ldexp(torch.ones_like(most), power), 1.0)


def _values(state, name):
    """What the FP8 codes stand for, exact in the rows' own type."""
    return (state[name].float() * state[name + "_scale"].transpose(2, 3)[..., None]).to(state["value"].dtype)


def _exact_norm_rope(case, state):
    d = case["head_dim"]
    cos, sin = state["cos"].double(), state["sin"].double()

    def turned(x, weight):
        x = x.double()
        x = x / ((x ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * weight.double()
        first, second = x.chunk(2, -1)
        c1, c2 = cos[:, None].chunk(2, -1)
        s1, s2 = sin[:, None].chunk(2, -1)
        return torch.cat((first * c1 - second * s1, second * c2 + first * s2), -1)

    out = [turned(state["query"], state["q_weight"])]
    for name, rows in (("k", turned(state["key"], state["k_weight"])), ("v", state["value"].double())):
        cache = state[name].double().contiguous()
        if case["cache"] == "fp8":  # the nearest of the row's 8-bit values, steps of a power of two
            step = 2.0 ** (rows.abs().amax(-1, keepdim=True) / 448.0).log2().ceil()
            rows = (rows / step).to(torch.float8_e4m3fn).double() * step
        cache.view(-1, case["kv_heads"], d)[state["slots"].long()] = rows
        out.append(cache)
    return tuple(out)


# --------------------------------------------------------------- page copies
def _prepare_copy(case, gen):
    shape = (case["layers"], case["blocks"], case["block"], case["kv_heads"], case["head_dim"])
    dtype = DTYPES[case["dtype"]]
    pages = torch.randperm(case["blocks"], generator=gen, device=DEVICE)[:2 * case["pairs"]].tolist()
    return {"k": torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype),
            "v": torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype),
            "src": pages[:case["pairs"]], "dst": pages[case["pairs"]:]}


def _plain_copy(state):
    src = torch.tensor(state["src"], device=DEVICE)
    dst = torch.tensor(state["dst"], device=DEVICE)
    state["k"][:, dst] = state["k"][:, src]
    state["v"][:, dst] = state["v"][:, src]
    return state["k"], state["v"]


# ----------------------------------------------------- the framework's calls
def _bind(case, state):
    """The handles that a serving loop keeps on its buffers."""
    import inferkernellab_amd as ikl

    if case["kind"] == "sample":
        one = {name: state[name] if case["mixed"] else case[name] for name in ("temperature", "top_k", "top_p", "min_p")}
        state["call"] = ikl.PreparedSampler(state["logits"], state["uniform"], logprobs=True, **one)
        return
    layers, blocks, block, kv_heads, head_dim = state["k"].shape
    cache = ikl.PagedKVCache(1, block, kv_heads, head_dim, num_layers=layers, dtype=state["k"].dtype, device=DEVICE,
                             act_dtype=DTYPES[case["dtype"]])
    cache.layout = ikl.CacheLayout(layers, blocks, block, kv_heads, head_dim)
    cache.k, cache.v = state["k"], state["v"]
    if "k_scale" in state:
        cache.k_scale, cache.v_scale = state["k_scale"], state["v_scale"]
    state["cache"] = cache
    if case["kind"] == "norm_rope":
        names = ("query", "key", "value", "q_weight", "k_weight", "cos", "sin")
        state["call"] = ikl.PreparedQKNormRopeAppend(*(state[n] for n in names), cache, state["slots"], eps=EPS,
                                                     query_out=state["query_out"])


def _own(state):
    kind = state["case"]["kind"]
    if kind == "sample":
        return dict(zip(("tokens", "policy", "sampling"), state["call"]()))
    if kind == "norm_rope":
        query_out = state["call"]()
        if "k_scale" in state:
            return query_out, _values(state, "k"), _values(state, "v")
        return query_out, state["k"], state["v"]
    import inferkernellab_amd as ikl

    ikl.copy_blocks_hip(state["cache"], state["src"], state["dst"])
    return state["k"], state["v"]
