"""4-bit weights that a caller lays out: their memory is their own. On the CPU."""

import pytest
import torch

from inferkernellab_amd import pack_int4_weight

ALIGNMENT = {"codes": 16, "scales": 16, "zeros": 4}  # bytes, of ikl_int4_linear


@pytest.mark.parametrize("group,cols", [(32, 128), (64, 128), (128, 128), (128, 256)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
def test_a_packed_weight_shares_no_memory_with_what_it_was_packed_from(group, cols, gated, offset):
    """A contraction of one step leaves the scales and zero points in the order
    that they were given in; a buffer's slice may start anywhere."""
    groups = cols // group
    codes = torch.randint(0, 16, (32, cols)).to(torch.uint8)
    scales = (torch.rand(offset + 32 * groups) + 0.5)[offset:].view(32, groups)
    zeros = torch.randint(0, 16, (offset + 32 * groups,), dtype=torch.uint8)[offset:].view(32, groups)
    w = pack_int4_weight(codes, scales, zeros, group_size=group, gated=gated)
    for name, of in ALIGNMENT.items():
        assert getattr(w, name).data_ptr() % of == 0, name
        assert getattr(w, name).is_contiguous()
    want = w.dequantize()
    for t in (codes, scales, zeros):
        t.zero_()
    assert torch.equal(w.dequantize(), want)
