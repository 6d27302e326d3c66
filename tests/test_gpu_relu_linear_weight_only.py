"""relu_linear8 where nothing needs the activations' gradient (a first layer's input, frozen layers before): none is formed, and what is, is the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_the_weight_alone(p, dtype):
    from bpt_amd import op
    rows, inner, outer = 2048, 2048, 64
    a, w, b = (torch.randn(s, device=DEV).to(dtype) for s in ((rows, inner), (outer, inner), (outer,)))
    do = torch.randn(rows, outer, device=DEV).to(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (a, w, b)]
    want = torch.autograd.grad(op.relu_linear8(*leaves, p, 5), leaves, do)[1:]
    leaves = [a, w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
    y = op.relu_linear8(*leaves, p, 5)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    got = torch.autograd.grad(y, leaves[1:], do)
    most = torch.cuda.max_memory_allocated() - held
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert most < 1.5 * a.numel() * a.element_size()              # the values of the codes, and results of a weight's size
