"""bias_table of the blocks' option bucket_bias: it starts at 0, also where reset_parameters draws the others."""
import pytest
import torch

from bpt_amd.block import BPTBlock, BPTMemBlock


@pytest.mark.parametrize("kind", [BPTBlock, BPTMemBlock])
def test_the_table_starts_at_0(kind):
    blk = kind(64, 2, 32, bucket_bias=7)
    assert not blk.bias_table.any()
    torch.nn.init.ones_(blk.bias_table)
    torch.manual_seed(3)
    blk.reset_parameters()
    assert not blk.bias_table.any() and blk.bias_table.requires_grad
    # the other parameters are drawn as those of a block without it
    plain = kind(64, 2, 32)
    torch.manual_seed(3)
    plain.reset_parameters()
    drawn = dict(blk.named_parameters())
    assert all(torch.equal(p, drawn[name]) for name, p in plain.named_parameters() if p.dim() > 1)
