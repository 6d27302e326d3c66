"""Which rows a block's norms hand to add_layer_norm: those that a workgroup's registers hold, 16 KiB, and float64's of any length.  The kernel holds the sum of
x and residual in 32 bits, torch's module has it rounded, and they add in other orders: their bits tell which ran."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("dtype,cols,kernel", [(torch.float32, 4096, True), (torch.float32, 4097, False), (torch.float32, 9000, False), (torch.bfloat16, 8192, True),
                                               (torch.bfloat16, 8193, False), (torch.float64, 2048, True), (torch.float64, 2049, True)])
def test_rows_around_16_kib(dtype, cols, kernel):
    from bpt_amd import op
    from bpt_amd.block import _add_norm
    gen = torch.Generator(device=DEV).manual_seed(cols)
    rand = lambda *s: torch.randn(s, generator=gen, device=DEV, dtype=torch.float64).to(dtype)
    norm = torch.nn.LayerNorm(cols, device=DEV, dtype=dtype)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * rand(cols)), norm.bias.copy_(rand(cols))
    x, r, dy = (rand(50, cols) for _ in range(3))
    leaves = [x, r, norm.weight, norm.bias]
    for t in leaves:
        t.requires_grad_(True)
    passes = [(y.detach(),) + torch.autograd.grad(y, leaves, dy)
              for y in (_add_norm(norm, x, r, True), op.add_layer_norm(x, r, norm.weight, norm.bias, norm.eps), norm(x + r))]
    same = [all(torch.equal(a, b) for a, b in zip(passes[0], other)) for other in passes[1:]]
    assert same == [kernel, not kernel]
