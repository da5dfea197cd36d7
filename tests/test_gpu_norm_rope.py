"""qk_norm_rope_append_kv_hip / PreparedQKNormRopeAppend on the GPU against
the formula in float64.

Tolerance: half a step of the output's type (``eps / 2`` of the value; fp16
below its normal range 2^-25), and the fp32 arithmetic before the rounding. A
lane sums 2N <= 16 squares and up to 6 partial sums follow, so the mean is off
by at most 24 half-steps of fp32 and its root by 12; the root's own step 2,
three products and a sum 4: below 20 x 2^-24 of |y1 cos| + |y2 sin|. FP8 rows:
half a step of E4M3 (2^-4 of the value, half its smallest value of 2^-9 times
the scale) and the same."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32_STEPS = 20 * 2.0 ** -24


def formula(x, w, cos, sin, eps):
    """(rotated rows, |y1 cos| + |y2 sin|) in float64."""
    x, w, cos, sin = (t.double() for t in (x, w, cos, sin))
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    half = x.shape[-1] // 2
    turned = torch.cat((-y[..., half:], y[..., :half]), -1)
    cos, sin = cos[:, None], sin[:, None]
    return y * cos + turned * sin, (y * cos).abs() + (turned * sin).abs()


def rounding(ref, dtype):
    floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return (ref.abs() * torch.finfo(dtype).eps / 2).clamp(min=floor)


def make(dtype, tokens, heads, kv, d, *, per_head=False, block=16, seed=0, fp8=False, layers=2, slot_dtype=torch.int32,
         head_major=None):
    from inferkernellab_amd.cache import PagedKVCache

    gen = torch.Generator().manual_seed(seed + tokens * 31 + d)
    blocks = -(-tokens // block) + 2

    def rows(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).cuda()

    angle = torch.rand(tokens, d, generator=gen) * 6.28
    cache = PagedKVCache(blocks, block, kv, d, num_layers=layers, device="cuda", head_major=head_major,
                         dtype=torch.float8_e4m3fn if fp8 else dtype, act_dtype=dtype if fp8 else None)
    for t in (cache.k, cache.v):
        t.copy_(torch.zeros(t.shape, device="cuda").to(t.dtype))
    slots = torch.randperm(blocks * block, generator=gen)[:tokens].to(slot_dtype).cuda()
    return dict(query=rows(tokens, heads, d, scale=3.0), key=rows(tokens, kv, d, scale=0.5), value=rows(tokens, kv, d),
                q_weight=rows(*((heads, d) if per_head else (d,)), scale=0.2, shift=1.0),
                k_weight=rows(*((kv, d) if per_head else (d,)), scale=0.2, shift=1.0), cos=angle.cos().to(dtype).cuda(),
                sin=angle.sin().to(dtype).cuda(), cache=cache, slots=slots)


def check(case, out, before, layer, eps, query_in, key_in):
    """Query rows, the layer's appended rows, and that nothing else changed."""
    cache, slots = case["cache"], case["slots"].long()
    dtype = query_in.dtype if query_in is not None else key_in.dtype
    if out is not None:
        ref, mag = formula(query_in, case["q_weight"], case["cos"], case["sin"], eps)
        assert ((out.double() - ref).abs() <= rounding(ref, dtype) + F32_STEPS * mag).all()
    ref, mag = formula(key_in, case["k_weight"], case["cos"], case["sin"], eps)
    bs = cache.layout.block_size
    ok = (slots >= 0) & (slots < cache.layout.num_blocks * bs)
    at = (layer, slots[ok] // bs, slots[ok] % bs)
    if cache.fp8:
        from inferkernellab_amd.cache import quantize_rows_e4m3
        scale = cache.k_scale[layer, at[1], :, at[2]].double()
        got = cache.k.float()[at].double() * scale[..., None]
        tol = (ref[ok].abs() * 2.0 ** -4).clamp(min=0) + 2.0 ** -10 * scale[..., None] + 2 * F32_STEPS * mag[ok]
        assert ((got - ref[ok]).abs() <= tol).all()
        most = ref[ok].abs().amax(-1)
        assert ((scale == 1) | ((scale >= most / 448 * (1 - 1e-5)) & (scale <= most / 224 * (1 + 1e-5)))).all()
        codes, vs = quantize_rows_e4m3(case["value"][ok])
        assert torch.equal(cache.v.view(torch.uint8)[at], codes.view(torch.uint8))
        assert torch.equal(cache.v_scale[layer, at[1], :, at[2]], vs)
    else:
        got = cache.k[at].double()
        assert ((got - ref[ok]).abs() <= rounding(ref[ok], dtype) + F32_STEPS * mag[ok]).all()
        assert torch.equal(cache.v[at], case["value"][ok])
    for now, old in zip((cache.k, cache.v), before):
        same = now.view(torch.uint8) == old.view(torch.uint8)
        same[at] = True
        assert same.all(), "a row outside the slots changed"


def run(case, layer=1, eps=1e-6, in_place=False, with_query=True):
    from inferkernellab_amd import qk_norm_rope_append_kv_hip

    cache = case["cache"]
    before = (cache.k.clone(), cache.v.clone())
    query = case["query"].clone() if with_query else None
    out = qk_norm_rope_append_kv_hip(query, case["key"], case["value"], case["q_weight"] if with_query else None,
                                     case["k_weight"], case["cos"], case["sin"], cache, case["slots"], layer, eps=eps,
                                     query_out=None if in_place or not with_query else torch.empty_like(query))
    torch.cuda.synchronize()
    if not with_query:
        assert out is None
    elif in_place:
        assert out is query
    else:
        assert torch.equal(query, case["query"])
    check(case, out, before, layer, eps, case["query"] if with_query else None, case["key"])
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv,d", [(1, 32, 8, 128), (2, 4, 2, 64), (7, 8, 1, 32), (33, 16, 4, 96),
                                               (19, 3, 3, 256), (5, 2, 1, 512), (130, 12, 12, 64), (3, 1, 1, 16),
                                               (70, 6, 2, 80)])
def test_against_the_formula(dtype, tokens, heads, kv, d):
    print(f"norm rope {dtype} T={tokens} H={heads}/{kv} D={d}", flush=True)
    run(make(dtype, tokens, heads, kv, d), in_place=tokens % 2 == 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv,d", [(1, 32, 8, 128), (33, 4, 2, 64), (517, 16, 4, 96), (9, 2, 1, 512),
                                               (300, 8, 8, 32)])
def test_into_the_fp8_cache(dtype, tokens, heads, kv, d):
    run(make(dtype, tokens, heads, kv, d, fp8=True))


@pytest.mark.parametrize("tokens,heads,kv", [(4096, 32, 8), (8193, 4, 1), (2049, 32, 32), (1025, 5, 5)])
def test_many_tokens(tokens, heads, kv):
    run(make(torch.bfloat16, tokens, heads, kv, 128))


def test_weights_per_head_slots_and_layouts():
    run(make(torch.bfloat16, 21, 8, 4, 128, per_head=True, slot_dtype=torch.int64))
    run(make(torch.float32, 21, 8, 4, 64, per_head=True, head_major=True, block=7))
    run(make(torch.float16, 21, 8, 4, 64, fp8=True, head_major=False, block=5), layer=0)
    run(make(torch.bfloat16, 40, 8, 4, 64), with_query=False)


def test_slots_outside_the_cache_are_skipped():
    for fp8 in (False, True):
        case = make(torch.bfloat16, 24, 8, 2, 128, fp8=fp8, slot_dtype=torch.int64)
        limit = case["cache"].layout.num_blocks * 16
        case["slots"][[0, 5, 9, 23]] = torch.tensor([-1, limit, 1 << 40, -(1 << 40)]).cuda()
        run(case)


@pytest.mark.parametrize("fp8", [False, True])
def test_offsets_past_32_bits(fp8):
    """The last pages of a cache of more than 4 GiB a tensor: the same rows as in a small one."""
    from inferkernellab_amd import qk_norm_rope_append_kv_hip
    from inferkernellab_amd.cache import PagedKVCache

    case = make(torch.bfloat16, 20, 8, 8, 128, fp8=fp8, layers=1)
    blocks = 280000 if fp8 else 140000
    bits = torch.uint8 if fp8 else torch.int16
    long = PagedKVCache(blocks, 16, 8, 128, num_layers=1, device="cuda", head_major=False,
                        dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16, act_dtype=torch.bfloat16 if fp8 else None)
    small = case["cache"]
    far = case["slots"] + (blocks - small.layout.num_blocks) * 16
    rows = [case[n] for n in ("query", "key", "value", "q_weight", "k_weight", "cos", "sin")]
    outs = [qk_norm_rope_append_kv_hip(rows[0].clone(), *rows[1:], cache, slots)
            for cache, slots in ((small, case["slots"]), (long, far))]
    assert torch.equal(*outs)
    for cache, slots in ((small, case["slots"]), (long, far)):
        at = (0, slots.long() // 16, slots.long() % 16)
        got = [cache.k.view(bits)[at], cache.v.view(bits)[at]]
        if fp8:
            got += [cache.k_scale[0, at[1], :, at[2]], cache.v_scale[0, at[1], :, at[2]]]
        if cache is small:
            want = got
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_strided_operands():
    """Columns of one fused projection, a misaligned view and transposed rows."""
    case = make(torch.bfloat16, 18, 8, 2, 64, seed=3)
    joined = torch.cat([case[n].reshape(18, -1) for n in ("query", "key", "value")], 1)
    case["key"] = joined[:, 512:640].view(18, 2, 64)
    case["value"] = joined[:, 640:].view(18, 2, 64)
    run(case)
    odd = torch.zeros(18 * 128 + 3, dtype=torch.bfloat16, device="cuda")
    odd[3:].copy_(case["key"].reshape(-1))
    case["key"] = odd[3:].view(18, 2, 64)
    case["cos"] = case["cos"].t().contiguous().t()
    case["k_weight"] = torch.cat((case["k_weight"][:1], case["k_weight"]))[1:]
    run(case)


def test_zero_rows_and_eps():
    case = make(torch.float32, 6, 2, 1, 64)
    case["key"][2] = 0
    case["query"][:] = 0
    run(case, eps=1e-5)
    case = make(torch.bfloat16, 6, 2, 1, 64, fp8=True)
    case["key"][2] = 0
    run(case, eps=1.0)
    case = make(torch.float32, 6, 2, 1, 64)
    case["key"] *= 1e-18                      # squares far below eps
    run(case)


def test_no_tokens():
    case = make(torch.bfloat16, 3, 4, 2, 64)
    for n in ("query", "key", "value", "cos", "sin", "slots"):
        case[n] = case[n][:0]
    assert run(case).shape == (0, 4, 64)


def test_prepared_streams_and_graphs():
    from inferkernellab_amd import PreparedQKNormRopeAppend

    case = make(torch.bfloat16, 32, 16, 4, 128, seed=5)
    cache, out = case["cache"], torch.empty_like(case["query"])
    names = ("query", "key", "value", "q_weight", "k_weight", "cos", "sin")
    call = PreparedQKNormRopeAppend(*(case[n] for n in names), cache, case["slots"], 1, query_out=out)
    before = (cache.k.clone(), cache.v.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert call() is out
    side.synchronize()
    check(case, out, before, 1, 1e-6, case["query"], case["key"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    for i in range(4):
        case["query"].copy_(torch.roll(case["query"], 1, 0))
        case["key"].mul_(1.5)
        out.zero_()
        graph.replay()
        (out.float().sum() * 2).item()
        check(case, out, before, 1, 1e-6, case["query"], case["key"])


def test_refusals():
    from inferkernellab_amd import PreparedQKNormRopeAppend, qk_norm_rope_append_kv_hip

    case = make(torch.bfloat16, 5, 4, 2, 64)
    names = ("query", "key", "value", "q_weight", "k_weight", "cos", "sin", "cache", "slots")

    def refused(error=ValueError, call=qk_norm_rope_append_kv_hip, **kw):
        args = {**case, **kw}
        rest = {k: v for k, v in args.items() if k not in names}
        with pytest.raises(error):
            call(*(args[n] for n in names), **rest)

    refused(key=case["key"][:, :1])
    refused(value=case["value"][:4])
    refused(cos=case["cos"][:, :32])
    refused(query=case["query"][:, :3])
    refused(query=case["query"].float())
    refused(q_weight=case["q_weight"][:32])
    refused(q_weight=case["q_weight"].float())
    refused(k_weight=case["k_weight"].repeat(3, 1))
    refused(k_weight=case["k_weight"].cpu())
    refused(slots=case["slots"][:4])
    refused(slots=case["slots"].float())
    refused(eps=-1.0)
    refused(eps=float("nan"))
    refused(query_out=case["query"][:4])
    refused(error=IndexError, layer=2)
    refused(call=PreparedQKNormRopeAppend, key=torch.stack((case["key"],) * 2, -1)[..., 0])
    refused(call=PreparedQKNormRopeAppend, slots=torch.stack((case["slots"],) * 2, -1)[:, 0])
