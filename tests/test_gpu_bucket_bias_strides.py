"""op.bucket_bias of tables and buckets that are not contiguous, both ways."""
import pytest
import torch

from bpt_amd import op

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_strided_tables_and_buckets(dtype):
    table = torch.randn(8, 11, device=DEV).to(dtype).t().requires_grad_(True)
    wide = torch.randint(0, 11, (200, 3), device=DEV)
    for buckets in (wide[:, 1], wide.view(-1)[::2], wide[:1, 0].expand(50)):
        assert not buckets.is_contiguous()
        bias = op.bucket_bias(table, buckets)
        assert torch.equal(bias, table[buckets])
        g = torch.randint(-4, 5, bias.shape, device=DEV).to(dtype)                 # (sums of few small whole numbers: exact)
        (dtable,) = torch.autograd.grad(bias, table, g.t().contiguous().t())
        assert torch.equal(dtable, torch.zeros_like(table).index_add(0, buckets, g))
