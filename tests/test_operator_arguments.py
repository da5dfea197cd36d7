"""Arguments of the normalised append, the page copies, the compaction and the
sampling that were taken wrongly or refused with another error."""

import pytest
import torch

from inferkernellab_amd import PagedKVCache, ops


def operands(tokens=3, heads=4, kv=2, d=32, device="cpu"):
    def rows(*shape):
        return torch.ones(*shape, device=device)

    cache = PagedKVCache(4, 4, kv, d, dtype=torch.float32, device=device)
    return [rows(tokens, heads, d), rows(tokens, kv, d), rows(tokens, kv, d), rows(d), rows(d), rows(tokens, d),
            rows(tokens, d), cache, torch.arange(tokens, dtype=torch.int32, device=device)]


@pytest.mark.parametrize("missing", [3, 4], ids=["q_weight", "k_weight"])
def test_a_missing_norm_weight_is_a_value_error(missing):
    args = operands()
    args[missing] = None
    with pytest.raises(ValueError, match="weight must have shape"):
        ops._qk_norm_rope_args(*args, 0, 1e-6, None)


@pytest.mark.parametrize("src,dst", [(bytes(8), [1] * 8), ([0] * 8, bytes(range(8))),
                                     (bytearray(range(8)), bytearray(range(8, 16))), (range(8), tuple(range(8, 16)))])
def test_block_ids_of_any_sequence_are_its_entries(src, dst):
    """Bytes are sequences of whole numbers too, not the memory of 64-bit ones."""
    for pairs, given in zip(ops._host_pairs(src, dst), (src, dst)):
        assert pairs.typecode == "q" and pairs.tolist() == list(given)


def test_block_ids_that_no_cache_has():
    for src, dst in (([1 << 70], [1]), ([1], [-(1 << 70)])):
        with pytest.raises(ValueError, match="invalid block id"):
            ops._host_pairs(src, dst)
    with pytest.raises(ValueError, match="one entry per copied block"):
        ops._host_pairs([1, 2], [3])
    for bad in ([1.5], ["1"], [None]):
        with pytest.raises(TypeError):
            ops._host_pairs(bad, [1])


def test_a_compaction_refuses_tables_it_cannot_change_in_place():
    """Before a page moves: after it, the tables that were not renumbered would name other requests' pages."""
    cache = PagedKVCache(8, 4, 2, 8)
    gone, first, second = cache.allocate_request(0, 8), cache.allocate_request(1, 8), cache.allocate_request(2, 8)
    cache.release_request(gone, 0)
    cache.k.copy_(torch.randn(cache.k.shape))
    before = cache.k.clone()
    for bad in (tuple(second), torch.tensor(second), range(4, 6)):
        with pytest.raises(ValueError, match="lists"):
            cache.compact([first, bad])
        assert (first, second) == ([2, 3], [4, 5]) and torch.equal(cache.k, before)
        assert cache.allocator.holders(2) == (1,) and cache.allocator.holders(4) == (2,)
    assert cache.compact(t for t in (first, second)) == {4: 0, 5: 1}
    assert (first, second) == ([2, 3], [0, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-44, 1e-46, 1e-300])
def test_a_temperature_below_float32_is_not_zero(temperature):
    """Its log probabilities are at that temperature (all mass on the likeliest tokens), not at 1."""
    from inferkernellab_amd import sample_tokens_hip

    logits = torch.randn(5, 1000, generator=torch.Generator().manual_seed(0))
    logits[3, [7, 70]] = 9.0
    for dtype in (torch.float32, torch.bfloat16):
        x = logits.to(dtype).cuda()
        x[[0, 1, 2, 4], [1, 2, 3, 4]] = 8.0
        uniform = torch.tensor([0.2, 0.5, 0.9, 0.75, 0.0]).cuda()
        for settings in (dict(), dict(min_p=0.5), dict(top_k=30, top_p=0.9)):
            tokens, policy, sampling = sample_tokens_hip(x, uniform, temperature=temperature, logprobs=True, **settings)
            want = torch.tensor([0.0, 0.0, 0.0, -0.6931471805599453, 0.0], dtype=torch.float64).float()
            assert tokens.tolist() == [1, 2, 3, 70, 4]
            assert torch.equal(policy.cpu(), want) and torch.equal(sampling.cpu(), want)
