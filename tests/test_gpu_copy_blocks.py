"""copy_blocks_hip on the GPU: the copied pages bit for bit in every layout
and type, and nothing else changed."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(dtype=torch.bfloat16, *, layers=3, blocks=40, block=16, kv=2, d=64, head_major=None, seed=0):
    from inferkernellab_amd.cache import PagedKVCache

    fp8 = dtype == torch.float8_e4m3fn
    cache = PagedKVCache(blocks, block, kv, d, num_layers=layers, dtype=dtype, device="cuda", head_major=head_major)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for t in (cache.k, cache.v) + ((cache.k_scale, cache.v_scale) if fp8 else ()):
        t.copy_(torch.randn(t.shape, generator=gen, device="cuda").to(t.dtype))
    return cache


def tensors(cache):
    return [cache.k, cache.v] + ([cache.k_scale, cache.v_scale] if cache.fp8 else [])


def bits(t):
    return t.contiguous().view(torch.uint8)


def check(cache, src, dst, **kw):
    from inferkernellab_amd import copy_blocks_hip

    want = [bits(t).clone() for t in tensors(cache)]
    as_list = [x.tolist() if isinstance(x, torch.Tensor) else list(x) for x in (src, dst)]
    limit = cache.layout.num_blocks
    for s, t in zip(*as_list):
        if 0 <= s < limit and 0 <= t < limit:
            for w in want:
                w[:, t] = w[:, s]
    assert copy_blocks_hip(cache, src, dst, **kw) is None
    torch.cuda.synchronize()
    for t, w in zip(tensors(cache), want):
        assert torch.equal(bits(t), w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("block,kv,d,layers", [(16, 2, 64, 3), (1, 1, 1, 2), (7, 3, 5, 1), (16, 8, 128, 2), (1, 1, 2, 4),
                                               (32, 4, 128, 1), (5, 2, 33, 2)])
def test_layouts_types_and_sizes(dtype, head_major, block, kv, d, layers):
    print(f"copy {dtype} head_major={head_major} page {block}x{kv}x{d} layers={layers}", flush=True)
    cache = make(dtype, layers=layers, blocks=12, block=block, kv=kv, d=d, head_major=head_major)
    check(cache, [3, 3, 0], [11, 7, 1])


@pytest.mark.parametrize("kind", [list, tuple, torch.int32, torch.int64])
@pytest.mark.parametrize("count", [0, 1, 2, 383, 384, 385, 900])
def test_lists_and_tensors(kind, count):
    cache = make(blocks=2000, layers=2, block=4, kv=1, d=16)
    pages = torch.randperm(2000, generator=torch.Generator().manual_seed(count))
    src, dst = pages[:count], pages[1000:1000 + count]
    if kind in (list, tuple):
        check(cache, kind(src.tolist()), kind(dst.tolist()))
    else:
        check(cache, src.to(kind).cuda(), dst.to(kind).cuda())
        check(cache, src.to(kind).cuda(), dst.to(kind).cuda().flip(0), validate_inputs=False)


def test_unchecked_tensors_skip_ids_outside():
    cache = make()
    src = torch.tensor([1, -1, 40, 2, 5], device="cuda")
    dst = torch.tensor([9, 10, 11, 40, 1 << 33], device="cuda")
    check(cache, src, dst, validate_inputs=False)
    check(cache, torch.arange(20, device="cuda")[::2], torch.arange(20, 40, device="cuda")[1::2])


def test_large_pages_and_many_layers():
    check(make(torch.float32, layers=32, blocks=30, block=32, kv=8, d=128), [0, 1, 2], [29, 20, 3])


def test_offsets_past_32_bits():
    """Pages of a layer that begin more than 2^32 bytes into the cache."""
    from inferkernellab_amd.cache import PagedKVCache
    from inferkernellab_amd import copy_blocks_hip

    cache = PagedKVCache(40000, 16, 8, 128, num_layers=4, dtype=torch.bfloat16, device="cuda")
    for t in (cache.k, cache.v):
        t[:, 39000].fill_(2.0)
        t[:, 39999].fill_(3.0)
        t[3, 39000].copy_(torch.randn(16, 8, 128).to(torch.bfloat16))
    copy_blocks_hip(cache, [39000], [39999])
    for t in (cache.k, cache.v):
        assert torch.equal(t[:, 39000], t[:, 39999]) and (t[0, 39999] == 2.0).all()


def test_streams_and_graphs():
    from inferkernellab_amd import copy_blocks_hip

    cache = make(blocks=64)
    src = torch.tensor([1, 2], device="cuda")
    dst = torch.tensor([30, 31], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        copy_blocks_hip(cache, [5], [6])
    side.synchronize()
    assert torch.equal(cache.k[:, 5], cache.k[:, 6])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        copy_blocks_hip(cache, src, dst, validate_inputs=False)  # read at each replay
        copy_blocks_hip(cache, [7, 8], [50, 51])                 # kept by the graph
    for i in range(4):
        cache.k.add_(1)
        src.copy_(torch.tensor([10 + i, 20 + i]))
        want_k, want_v = bits(cache.k).clone(), bits(cache.v).clone()
        for w in (want_k, want_v):
            w[:, [30, 31, 50, 51]] = w[:, [10 + i, 20 + i, 7, 8]]
        graph.replay()
        cache.k.float().sum().item()
        assert torch.equal(bits(cache.k), want_k) and torch.equal(bits(cache.v), want_v)


def test_refusals():
    from inferkernellab_amd import copy_blocks_hip
    from inferkernellab_amd.cache import PagedKVCache

    cache = make()
    before = bits(cache.k).clone()

    def both(src, dst, message):
        with pytest.raises(ValueError, match=message):
            copy_blocks_hip(cache, src, dst)
        with pytest.raises(ValueError, match=message):
            copy_blocks_hip(cache, torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda"))

    both([0], [40], "invalid block id")
    both([-1], [1], "invalid block id")
    both([0, 1], [5, 5], "written twice")
    both([0, 1], [1, 2], "read and written")
    both([0, 1], [2], "one entry per copied block")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    for src, dst in (([1], one), (one, one.long()), (one.float(), one.float()), (one.cpu(), one.cpu()), (one[None], one[None])):
        with pytest.raises(ValueError):
            copy_blocks_hip(cache, src, dst)
    with pytest.raises(TypeError):
        copy_blocks_hip(cache, [1.5], [2])
    with pytest.raises(ValueError, match="GPU"):
        copy_blocks_hip(PagedKVCache(4, 4, 1, 8), [0], [1])
    assert torch.equal(bits(cache.k), before)
