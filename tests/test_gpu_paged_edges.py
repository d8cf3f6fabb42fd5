"""The operators of the paged KV cache at the ends of what they accept."""
import pytest
import torch

import fstattention_amd as fsta

pytestmark = pytest.mark.gpu


def test_masks_wider_than_32_bits_count():
    """64 nodes of 2^25 words: the words of a workgroup's rows are 2^31 in number.  Memory that held something else before."""
    nodes, most = 64, 1 << 30
    dirty = torch.full((nodes, most // 32), -1, dtype=torch.int32, device="cuda")
    del dirty
    bits = fsta.tree_mask_bits(torch.arange(-1, nodes - 1).cuda(), torch.tensor([0, nodes], dtype=torch.int32).cuda(), most)
    assert bits.shape == (nodes, most // 32)
    chain = [(2 << i) - 1 for i in range(nodes)]
    signed = lambda x: x - (1 << 32) if x >> 31 else x
    assert bits[:, :2].tolist() == [[signed(x & 0xffffffff), signed(x >> 32)] for x in chain]
    for row in bits:
        assert int(row[2:].count_nonzero()) == 0


@pytest.mark.parametrize("most", [-1, 1 << 31, 1 << 37])
def test_more_nodes_than_a_tree_can_have_are_refused(most):
    """2^37 nodes are 2^32 words, which the library's 32-bit count would take for none."""
    with pytest.raises(ValueError, match="max_nodes"):
        fsta.tree_mask_bits(torch.zeros(1, dtype=torch.int64).cuda(), max_nodes=most)
