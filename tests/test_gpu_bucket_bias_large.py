"""op.bucket_bias of more elements than a launch has threads."""
import pytest
import torch

from bpt_amd import op

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("n_edges,heads", [(2 ** 26, 64), (2 ** 26 + 3, 65), (2 ** 22 + 1, 1024)])
def test_scores_of_many_edges(n_edges, heads):
    """Rows that share a bucket are equal, and those of the table: in pieces, the last edges among them."""
    n = 7
    table = torch.randn(n, heads, dtype=torch.bfloat16, device=DEV)
    buckets = torch.arange(n_edges, device=DEV) % (n + 1)                         # (n: outside of the table)
    rows = torch.cat([table, torch.zeros(1, heads, dtype=torch.bfloat16, device=DEV)])
    bias = op.bucket_bias(table, buckets)
    assert bias.shape == (n_edges, heads) and bias.numel() >= 2 ** 32
    for first in list(range(0, n_edges, 2 ** 24 - 1)) + [n_edges - 100]:
        part = slice(first, min(first + 2 ** 20, n_edges))
        assert torch.equal(bias[part], rows[buckets[part]]), first
