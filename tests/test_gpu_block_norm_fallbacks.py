"""A block's norms with parameters that the kernels have no rules for (tangents, subclasses of Tensor): torch's module runs, as it did before there were kernels."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def block(**kw):
    from bpt_amd.block import BPTBlock
    torch.manual_seed(1)
    return BPTBlock(64, 4, 128, drop_h=0.0, drop_a=0.0, **kw).to(DEV)


@pytest.mark.parametrize("which", ["weight", "bias"])
def test_a_tangent_of_a_norms_parameter(which):
    """d/dt of norm(x + r) along a tangent t of weight (bias) is xhat t (t): the torch module has it."""
    from bpt_amd.block import _add_norm
    norm = block().norm_inter
    x, r, t = torch.randn(20, 64, device=DEV), torch.randn(20, 64, device=DEV), torch.randn(64, device=DEV)
    kept = getattr(norm, which)
    with fwAD.dual_level():
        delattr(norm, which)
        setattr(norm, which, fwAD.make_dual(kept.detach(), t))
        tangent = fwAD.unpack_dual(_add_norm(norm, x, r, True)).tangent
    z = (x + r).double()
    xhat = (z - z.mean(1, keepdim=True)) / torch.sqrt(z.var(1, unbiased=False, keepdim=True) + norm.eps)
    want = xhat * t.double() if which == "weight" else t.double().expand(20, 64)
    assert (tangent.double() - want).abs().max() <= 1e-5 * want.abs().max()


class Marked(torch.Tensor):
    """A tensor with rules of its own: counts the functions that are called on it."""
    calls = 0

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        Marked.calls += func is torch.nn.functional.layer_norm
        return super().__torch_function__(func, types, args, kwargs or {})


def test_a_norms_parameter_of_a_subclass():
    from bpt_amd.block import _add_norm
    norm = block().norm_inter
    x, r = torch.randn(20, 64, device=DEV), torch.randn(20, 64, device=DEV)
    want, weight = _add_norm(norm, x, r, True), norm.weight
    del norm.weight
    norm.weight = weight.detach().as_subclass(Marked)
    Marked.calls = 0
    got = _add_norm(norm, x, r, True)
    assert Marked.calls == 1 and (got.as_subclass(torch.Tensor) - want).abs().max() < 1e-5
