"""The largest launch: HIP takes fewer than 2^32 threads of a grid. What does
not fit is refused on the host, before anything is launched."""

import ctypes

import pytest
import torch

from inferkernellab_amd import _lib
from tests.test_new_operator_refusals import _copy, _norm_rope, _sample


@pytest.mark.parametrize("layers,page,status", [((1 << 24) // 2, 4096, _lib.IKL_EINVAL),
                                                ((1 << 24) // 4, 2 * 16 * 1024, _lib.IKL_EINVAL)])
def test_copy_refuses_one_page_that_no_launch_holds(layers, page, status):
    """2 tensors of 2^23 layers, a workgroup each, and of 2^22 layers, two each: 2^24 workgroups of 256."""
    a, keep = _copy([0], [1], num_layers=layers)
    for n in range(2):
        a.page_bytes[n] = page
    assert _lib.load().ikl_copy_blocks(ctypes.byref(a), None) == status
    assert "too many pages" in _lib.last_error()


@pytest.mark.parametrize("rows", [1 << 22, 1 << 30])
def test_sample_refuses_rows_that_no_launch_holds(rows):
    """A workgroup of 1024 a row."""
    assert _lib.load().ikl_sample_tokens(ctypes.byref(_sample(rows=rows)), None) == _lib.IKL_EINVAL
    assert "too many rows" in _lib.last_error()


@pytest.mark.parametrize("head_dim,tokens", [(64, 1 << 27), (128, 1 << 26), (512, 1 << 24), (1024, (1 << 31) - 1)])
def test_norm_rope_refuses_rows_that_no_launch_holds(head_dim, tokens):
    """8 rows a token in workgroups of 64, 32 or 8 rows (bf16 heads of 64, 128, 512): 2^24 workgroups of 256."""
    args = _norm_rope(num_tokens=tokens, head_dim=head_dim)
    assert _lib.load().ikl_qk_norm_rope_append_kv(ctypes.byref(args), None) == _lib.IKL_EINVAL
    assert "too many rows" in _lib.last_error()


@pytest.mark.gpu
def test_sample_of_the_most_rows_a_launch_holds():
    from inferkernellab_amd import sample_tokens_hip

    rows = (1 << 22) - 1
    logits = torch.randint(0, 2, (rows, 2), device="cuda").to(torch.bfloat16)
    tokens = sample_tokens_hip(logits, torch.full((rows,), 0.999999, device="cuda"), temperature=0.0)
    assert torch.equal(tokens, (logits[:, 1] > logits[:, 0]).long())
    with pytest.raises(ValueError, match="too many rows"):
        sample_tokens_hip(logits[:1].expand(rows + 1, -1), torch.zeros(rows + 1, device="cuda"))


@pytest.mark.gpu
def test_copies_of_more_pages_than_one_launch_holds():
    """4.3 million pairs of 2 layers, 17 million workgroups: in two launches."""
    from inferkernellab_amd import PagedKVCache, copy_blocks_hip

    pairs = (1 << 22) + 100001
    cache = PagedKVCache(2 * pairs, 1, 1, 8, num_layers=2, dtype=torch.bfloat16, device="cuda")
    for t in (cache.k, cache.v):
        t.view(torch.int16).copy_(torch.randint(-30000, 30000, t.shape, dtype=torch.int16, device="cuda"))
    order = torch.randperm(2 * pairs, device="cuda")
    src, dst = order[:pairs].to(torch.int32), order[pairs:].to(torch.int32)
    want = [t.view(torch.int16)[:, order[:pairs]] for t in (cache.k, cache.v)]
    copy_blocks_hip(cache, src, dst, validate_inputs=False)
    for t, w in zip((cache.k, cache.v), want):
        assert torch.equal(t.view(torch.int16)[:, order[pairs:]], w)
        assert torch.equal(t.view(torch.int16)[:, order[:pairs]], w)
