"""sample_tokens_hip / PreparedSampler on the GPU against the definition in
numpy float64: the tokens have to be the same. A token differs from the
definition's only where the uniform number's share of the mass lies within
the masses' error of a border, vocab x 2^-(bits+1) of the likeliest weight
(below 2^-29 at 131072 tokens); the fixed seeds here have no such case. Log
probabilities are rounded once to float32 from doubles: half a step of the
value, and 2^-28 for the masses."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def oracle_row(x, u, t, k, p, q):
    """(token, policy, sampling) of one row by the definition."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, -np.inf, -np.inf
    greedy = not t > 0
    order = np.argsort(-x, kind="stable")
    s = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        logw = np.where(s == s[0], 0.0, (s - s[0]) / (1.0 if greedy else t))
    logw = np.where(s == -np.inf, -np.inf, logw)
    w = np.exp(logw)
    n = k if 0 < k < len(x) else len(x)
    before = np.concatenate(([0.0], np.cumsum(w)))
    if p < 1:
        n = min(n, int((before[:n] <= max(p, 0.0) * before[n]).sum()))
    if q > 0:
        n = min(n, int((w >= min(q, 1.0)).sum()))
    aim = (0.0 if greedy else u) * before[n]
    at = int((before[1:n + 1] <= aim).sum())
    at = min(at, int((w[:n] > 0).sum()) - 1)
    return int(order[at]), logw[at] - np.log(before[-1]), logw[at] - np.log(before[n])


def per_row(value, rows):
    return value.double().cpu().numpy() if isinstance(value, torch.Tensor) else np.full(rows, np.float32(value))


def check(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, got=None):
    from inferkernellab_amd import sample_tokens_hip

    if got is None:
        got = sample_tokens_hip(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                                logprobs=True)
    tokens, policy, sampling = (t.cpu().numpy() for t in got)
    rows = logits.shape[0]
    assert tokens.dtype == np.int64 and policy.dtype == sampling.dtype == np.float32
    t, k, p, q = (per_row(v, rows) for v in (temperature, top_k, top_p, min_p))
    x, u = logits.float().cpu().numpy(), uniform.cpu().numpy().astype(np.float64)
    for b in range(rows):
        want, lp, ls = oracle_row(x[b], u[b], float(t[b]), int(k[b]), float(p[b]), float(q[b]))
        assert tokens[b] == want, (b, tokens[b], want)
        for g, w in ((policy[b], lp), (sampling[b], ls)):
            assert g == w or abs(g - w) <= 2.0 ** -24 * abs(w) + 2.0 ** -28, (b, g, w)


def inputs(rows, vocab, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=gen) * spread
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 20), generator=gen), torch.rand(rows, 20, generator=gen) * 9)
    return x.to(DTYPES[dtype]).cuda(), torch.rand(rows, generator=gen).cuda()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 64, 65, 255, 1000, 8191, 32000, 50257])
@pytest.mark.parametrize("settings", [dict(), dict(temperature=0.7, top_p=0.9), dict(top_k=50, top_p=0.95),
                                      dict(temperature=1.5, top_k=7, min_p=0.05), dict(temperature=0.0, top_p=0.5)],
                         ids=["all", "topp", "topk_topp", "topk_minp", "greedy"])
def test_tokens_and_logprobs(vocab, dtype, settings):
    rows = 3 if vocab > 10000 else 9
    print(f"sample rows={rows} vocab={vocab} {dtype} {settings}", flush=True)
    logits, uniform = inputs(rows, vocab, dtype, vocab * 7 + len(settings))
    check(logits, uniform, **settings)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [4093, 4095, 4096, 4097, 8185, 8190, 8192, 8193, 8199, 12287, 16385, 24583, 32769,
                                   40961])
def test_rows_that_end_near_a_round_of_the_threads(vocab, dtype):
    """Rows of odd lengths one behind the other start at every alignment."""
    logits, uniform = inputs(9, vocab, dtype, vocab)
    check(logits, uniform)
    check(logits, uniform, top_k=40, top_p=0.9)
    check(logits, uniform, min_p=0.01)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,vocab", [(1, 131072), (5, 131072), (300, 4001), (2, 400003)])
def test_large_rows(rows, vocab, dtype):
    logits, uniform = inputs(rows, vocab, dtype, rows)
    check(logits, uniform, temperature=1.1, top_p=0.97, min_p=0.001)
    check(logits, uniform, temperature=1.1)


@pytest.mark.parametrize("top_k", [1, 2, 100, 1000, 31999, 32000, 40000])
def test_top_k_range(top_k):
    logits, uniform = inputs(4, 32000, "bf16", 3)
    check(logits, uniform, top_k=top_k, top_p=0.999)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.3, 30.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_flat_and_steep_rows(spread, dtype):
    gen = torch.Generator().manual_seed(4)
    logits = (torch.randn(4, 20011, generator=gen) * spread).to(DTYPES[dtype]).cuda()
    uniform = torch.rand(4, generator=gen).cuda()
    check(logits, uniform, top_p=0.9)
    check(logits, uniform, top_k=9000, top_p=0.5)
    check(logits, uniform)


def test_equal_logits_have_exact_borders():
    """n equal logits weigh 1 each: every mass is a whole number, and so exact."""
    logits = torch.full((8, 64), -3.25).cuda()
    uniform = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.984375, 0.96875, 0.1, 0.99999994]).cuda()
    check(logits, uniform)
    check(logits, uniform, top_p=0.5)   # the token with exactly half before it is kept
    check(logits, uniform, top_k=16, top_p=0.25)
    check(logits, uniform, min_p=1.0)
    from inferkernellab_amd import sample_tokens_hip
    assert sample_tokens_hip(logits, uniform).tolist() == [0, 16, 32, 48, 63, 62, 6, 63]


def test_ties_at_the_cuts():
    """Few distinct values, so that every cut falls inside a group of equal logits."""
    gen = torch.Generator().manual_seed(5)
    logits = torch.randint(0, 6, (16, 4099), generator=gen).to(torch.bfloat16).cuda()
    uniform = torch.rand(16, generator=gen).cuda()
    for settings in (dict(top_k=100), dict(top_p=0.4), dict(top_k=900, top_p=0.8), dict(min_p=0.1), dict()):
        check(logits, uniform, temperature=1.25, **settings)


def test_masked_and_odd_values():
    inf, nan = float("inf"), float("nan")
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(12, 777, generator=gen) * 2
    x[0] = -inf                                # nothing to draw
    x[1] = nan
    x[2, 5:] = -inf
    x[3] = -inf
    x[3, 776] = -1e30                          # one token left
    x[4, ::2] = nan
    x[5, [10, 200, 700]] = inf                 # share all mass
    x[6] = torch.finfo(torch.float32).min      # a mask of the lowest value all over
    x[7, 1:] = torch.finfo(torch.float32).min
    x[8] = 0.0
    x[8, ::2] = -0.0                           # equal to 0
    x[9] = 1e-42                               # subnormal
    x[10, :] = inf
    uniform = torch.rand(12, generator=gen).cuda()
    for settings in (dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.0),
                     dict(temperature=1e-30), dict(temperature=1e30, top_p=0.6)):
        print(settings, flush=True)
        check(x.cuda(), uniform, **settings)
    half = x.to(torch.float16).cuda()
    check(half, uniform, top_k=5, top_p=0.9)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [24576, 24577, 40003])
def test_masked_and_odd_values_of_long_rows(vocab, dtype):
    """The same on both sides of the length from which rows are split, with NaN, masks and infinities in some
    workgroups' parts only."""
    inf, nan = float("inf"), float("nan")
    gen = torch.Generator().manual_seed(17)
    low = torch.finfo(DTYPES[dtype]).min
    x = torch.randn(14, vocab, generator=gen) * 2
    x[0] = -inf
    x[1] = nan
    x[2, 5:] = -inf
    x[3] = -inf
    x[3, vocab - 1] = -1e30
    x[4, ::2] = nan
    x[5, [10, vocab // 2, vocab - 1]] = inf
    x[6] = low
    x[7, 1:] = low
    x[8] = 0.0
    x[8, ::2] = -0.0
    x[9, :vocab // 2] = -inf
    x[10] = inf
    x[11, :vocab - 3000] = nan
    x[12] = (torch.randint(0, 6, (vocab,), generator=gen)).float()   # ties at every cut
    x[13] = 1e4                                                      # one heavy token among equal ones
    x[13, vocab // 3] = 1e4 + 64
    logits = x.to(DTYPES[dtype]).cuda()
    uniform = torch.rand(14, generator=gen).cuda()
    for settings in (dict(), dict(top_k=3), dict(top_k=3000, top_p=0.7), dict(top_p=0.7), dict(min_p=0.2),
                     dict(top_p=0.9, min_p=0.01), dict(top_k=500, min_p=0.01), dict(top_k=20000, top_p=0.8, min_p=0.05),
                     dict(min_p=1.0), dict(temperature=0.0), dict(temperature=1e-30),
                     dict(temperature=1e30, top_p=0.6)):
        print(vocab, dtype, settings, flush=True)
        check(logits, uniform, **settings)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.3, 30.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_flat_and_steep_long_rows(spread, dtype):
    gen = torch.Generator().manual_seed(18)
    logits = (torch.randn(3, 40009, generator=gen) * spread).to(DTYPES[dtype]).cuda()
    uniform = torch.rand(3, generator=gen).cuda()
    for settings in (dict(), dict(top_p=0.9), dict(top_k=9000, top_p=0.5), dict(min_p=0.9),
                     dict(top_k=9000, min_p=0.5)):
        print(spread, dtype, settings, flush=True)
        check(logits, uniform, **settings)


@pytest.mark.parametrize("vocab", [20011, 40009])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257, 511, 513, 1025, 2047, 2048, 2049])
def test_tokens_crowded_in_one_step_of_the_histogram(n, vocab):
    """n distinct logits within 1/5000 of the row's range, so that every cut falls among all of them."""
    gen = torch.Generator().manual_seed(n + vocab)
    x = torch.full((4, vocab), float("-inf"))
    for row in x:
        at = torch.randperm(vocab, generator=gen)[:n + 3]
        row[at[:n]] = 5 + 2e-6 * torch.arange(n)
        row[at[n:]] = -15.0
    uniform = torch.rand(4, generator=gen).cuda()
    for settings in (dict(), dict(top_p=0.37), dict(top_k=n // 2 + 1), dict(top_k=n // 2 + 1, top_p=0.61),
                     dict(top_p=0.8, min_p=0.5), dict(top_k=n // 3 + 1, top_p=0.9, min_p=0.9995)):
        print(n, vocab, settings, flush=True)
        check(x.cuda(), uniform, **settings)


@pytest.mark.parametrize("min_p", [0.02, 0.005, 0.002, 1e-3, 1e-4, 1e-8, 1e-20])
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_min_p_of_many_candidates(min_p, dtype):
    """Some hundred to all of 20011 tokens are candidates."""
    gen = torch.Generator().manual_seed(25)
    logits = (torch.randn(5, 20011, generator=gen) * 2).to(DTYPES[dtype]).cuda()
    uniform = torch.rand(5, generator=gen).cuda()
    for settings in (dict(), dict(top_p=0.9), dict(top_k=700)):
        print(min_p, dtype, settings, flush=True)
        check(logits, uniform, min_p=min_p, **settings)


def test_long_rows_with_settings_per_row_and_strides():
    rows = 20
    base, uniform = inputs(rows, 60100, "fp16", 19)
    gen = torch.Generator().manual_seed(20)

    def pick(values, dtype=torch.float32):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (rows,), generator=gen)].cuda()

    for view in (base[:, 3:50260], base[:, :50257], base[2:3, 1:50002].expand(rows, -1)):
        check(view, uniform, temperature=pick([0.0, 0.5, 1.0, 2.0]), top_k=pick([0, 1, 30, 3000, 99999], torch.int64),
              top_p=pick([1.0, 0.9, 0.2]), min_p=pick([0.0, 0.001, 0.3, 1.0]))


def test_one_sampler_on_rows_that_change_kind():
    """A workspace keeps nothing: the same split rows drawn from, then masked, then infinite, then drawn from again."""
    from inferkernellab_amd import PreparedSampler
    base, uniform = inputs(2, 50257, "bf16", 21)
    logits = base.clone()
    call = PreparedSampler(logits, uniform, top_p=0.9, min_p=0.01, logprobs=True)
    for fill in (None, float("-inf"), 0.0, None, float("inf"), float("nan"), None):
        logits.copy_(base) if fill is None else logits.fill_(fill)
        check(logits, uniform, top_p=0.9, min_p=0.01, got=call())


def test_more_rows_than_a_grid_dimension_of_16_bits():
    gen = torch.Generator().manual_seed(22)
    logits = torch.randn(70001, 3, generator=gen).cuda()
    uniform = torch.rand(70001, generator=gen).cuda()
    from inferkernellab_amd import sample_tokens_hip
    got = sample_tokens_hip(logits, uniform, logprobs=True)
    check(logits[-50:], uniform[-50:], got=[t[-50:] for t in got])


def test_eager_call_inside_a_capture():
    from inferkernellab_amd import sample_tokens_hip
    logits, uniform = inputs(4, 50257, "bf16", 23)
    sample_tokens_hip(logits, uniform, top_k=20)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        got = sample_tokens_hip(logits, uniform, top_k=20, logprobs=True)
    gen = torch.Generator().manual_seed(24)
    for _ in range(4):
        uniform.copy_(torch.rand(4, generator=gen))
        logits.copy_(torch.roll(logits, 1001, 1))
        g.replay()
        (logits.float().sum()).item()
        check(logits, uniform, top_k=20, got=got)


def test_settings_per_row_and_out_of_range():
    rows = 24
    logits, uniform = inputs(rows, 5003, "fp16", 8)
    gen = torch.Generator().manual_seed(9)

    def pick(values, dtype=torch.float32):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (rows,), generator=gen)].cuda()

    for wide in (torch.int32, torch.int64):
        check(logits, uniform, temperature=pick([0.0, 0.5, 1.0, 2.0]), top_k=pick([0, 1, 30, 5003, 9999], wide),
              top_p=pick([1.0, 0.9, 0.2]), min_p=pick([0.0, 0.3, 1.0]))
    # tensors are not looked at on the host: the nearest value with a meaning
    nan, inf = float("nan"), float("inf")
    check(logits, uniform, temperature=pick([-1.0, nan, 1.0]), top_k=pick([-5, 0, 7], torch.int64),
          top_p=pick([2.0, inf, 0.0, -3.0]), min_p=pick([-1.0, 7.0, 0.0]))
    from inferkernellab_amd import sample_tokens_hip
    hot = sample_tokens_hip(logits, torch.full((rows,), 1.5).cuda())
    last = sample_tokens_hip(logits, torch.full((rows,), 0.99999994).cuda())
    assert torch.equal(hot, last)
    cold = sample_tokens_hip(logits, torch.full((rows,), nan).cuda())
    assert torch.equal(cold, logits.float().argmax(-1))


def test_strided_and_misaligned_rows():
    gen = torch.Generator().manual_seed(10)
    base = (torch.randn(7, 3100, generator=gen) * 2).cuda()
    uniform = torch.rand(14, generator=gen).cuda()[::2]
    for dtype in DTYPES.values():
        for view in (base.to(dtype)[:, 3:3002], base.to(dtype)[:, 1::3], base.to(dtype).t().contiguous().t(),
                     base.to(dtype)[1:2].expand(7, -1)):
            check(view, uniform, top_k=300, top_p=0.9)


def test_results_do_not_depend_on_neighbours():
    """A row draws the same alone, in a batch, and at another place of it."""
    from inferkernellab_amd import sample_tokens_hip
    logits, uniform = inputs(40, 50257, "bf16", 11)
    whole = sample_tokens_hip(logits, uniform, top_p=0.9, logprobs=True)
    for b in (0, 17, 39):
        one = sample_tokens_hip(logits[b:b + 1], uniform[b:b + 1], top_p=0.9, logprobs=True)
        for x, y in zip(whole, one):
            assert torch.equal(x[b:b + 1], y)


def test_no_rows_and_tokens_only():
    from inferkernellab_amd import sample_tokens_hip
    logits, uniform = inputs(6, 900, "bf16", 12)
    assert sample_tokens_hip(logits[:0], uniform[:0]).shape == (0,)
    tokens = sample_tokens_hip(logits, uniform, temperature=0.8)
    assert torch.equal(tokens, sample_tokens_hip(logits, uniform, temperature=0.8, logprobs=True)[0])


def test_prepared_on_streams_and_in_graphs():
    """Two samplers on two streams, and captured: every replay equals the eager call on the buffers' new values."""
    from inferkernellab_amd import PreparedSampler, sample_tokens_hip
    a, ua = inputs(8, 32000, "bf16", 13)
    b, ub = inputs(3, 50257, "fp32", 14)
    one = PreparedSampler(a, ua, temperature=0.8, top_p=0.9, logprobs=True)
    two = PreparedSampler(b, ub, top_k=40)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, call in zip(streams, (one, two)):
            with torch.cuda.stream(s):
                call()
    torch.cuda.synchronize()
    check(a, ua, temperature=0.8, top_p=0.9, got=(one.tokens, one.policy_logprobs, one.sampling_logprobs))
    assert torch.equal(two.tokens, sample_tokens_hip(b, ub, top_k=40))
    graphs = []
    for call in (one, two):
        with torch.cuda.stream(streams[0]):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[0]):
                call()
            graphs.append(g)
    gen = torch.Generator().manual_seed(15)
    for i in range(4):
        a.copy_(torch.roll(a, 77, 1))
        ua.copy_(torch.rand(8, generator=gen))
        ub.copy_(torch.rand(3, generator=gen))
        for g in graphs:
            g.replay()
        (a.float() @ a.float().t()).sum().item()  # other work and a wait between the replays
        check(a, ua, temperature=0.8, top_p=0.9, got=(one.tokens, one.policy_logprobs, one.sampling_logprobs))
        assert torch.equal(two.tokens, sample_tokens_hip(b, ub, top_k=40)), i


def test_refusals():
    from inferkernellab_amd import PreparedSampler, sample_tokens_hip
    logits, uniform = inputs(4, 100, "fp32", 16)
    for bad, message in ((dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                         (dict(top_k=-1), "top_k"), (dict(top_k=1.5), "top_k"), (dict(top_k=float("inf")), "top_k"),
                         (dict(top_p=0.0), "top_p"),
                         (dict(top_p=1.1), "top_p"), (dict(min_p=-0.1), "min_p"), (dict(min_p=1.1), "min_p"),
                         (dict(top_k=torch.ones(4).cuda()), "top_k"), (dict(top_p=torch.ones(3).cuda()), "top_p"),
                         (dict(min_p=torch.ones(4)), "min_p"),
                         (dict(temperature=torch.ones(4, dtype=torch.float64).cuda()), "temperature")):
        with pytest.raises(ValueError, match=message):
            sample_tokens_hip(logits, uniform, **bad)
    for bad in (logits[0], logits.cpu(), logits.double(), logits.int(), logits[:, :0]):
        with pytest.raises(ValueError):
            sample_tokens_hip(bad, uniform)
    for bad in (uniform[:3], uniform.cpu(), uniform.double(), uniform[None]):
        with pytest.raises(ValueError, match="uniform"):
            sample_tokens_hip(logits, bad)
    with pytest.raises(ValueError, match="contiguous"):
        PreparedSampler(logits.t().contiguous().t(), uniform)
