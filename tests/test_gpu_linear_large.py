"""op.linear_act of as many columns as it takes."""
import pytest
import torch

from bpt_amd import op

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("outer", [2 ** 24 + 5, 2 ** 28])
def test_gradients_of_many_columns(outer):
    """y = 3 w + b of two rows; the gradients are those of small whole numbers, exact."""
    x = torch.tensor([[3.0], [5.0]], device=DEV)
    w = (torch.arange(outer, device=DEV) % 1000).float().view(-1, 1).requires_grad_(True)
    b = (torch.arange(outer, device=DEV) % 7).float().requires_grad_(True)
    y = op.linear_act(x, w, b)
    assert torch.equal(y[0], 3 * w[:, 0] + b) and torch.equal(y[1], 5 * w[:, 0] + b)
    dy = (torch.arange(outer, device=DEV) % 11).float()
    dw, db = torch.autograd.grad(y, (w, b), torch.stack([dy, 2 * dy]))
    assert torch.equal(db, 3 * dy) and torch.equal(dw[:, 0], 13 * dy)
