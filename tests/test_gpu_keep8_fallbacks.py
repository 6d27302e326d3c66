"""Feed-forwards with keep8 in calls that relu_linear8 has no form for: they compute what they do without keep8."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


class Marked(torch.Tensor):
    """A tensor with rules of its own."""


def ffn(dtype=torch.float32, keep8=True, dropout=0.0):
    from bpt_amd.block import PositionwiseFeedForward
    torch.manual_seed(2)
    return PositionwiseFeedForward(64, 128, dropout, keep8=keep8).to(DEV, dtype)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float16])
def test_feed_forward_of_other_types(dtype):
    x = torch.randn(30, 64, device=DEV, dtype=dtype, requires_grad=True)
    got = [m(x) for m in (ffn(dtype), ffn(dtype, keep8=False))]
    assert got[0].dtype == dtype and torch.equal(*got)
    grads = [torch.autograd.grad(y.sum(), x)[0] for y in got]
    assert torch.equal(*grads)


def test_feed_forward_inside_autocast_to_float16():
    x = torch.randn(30, 64, device=DEV, requires_grad=True)
    with torch.autocast("cuda"):
        got = [m(x) for m in (ffn(), ffn(keep8=False))]
    assert got[0].dtype == torch.float16 and torch.equal(*got)
    assert torch.equal(*(torch.autograd.grad(y.float().sum(), x)[0] for y in got))


def test_feed_forward_inside_autocast_to_bfloat16_keeps_8_bits():
    x = torch.randn(30, 64, device=DEV, requires_grad=True)
    m, kept = ffn(), []
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.dtype) or t, lambda t: t):
        y = m(x)
    assert y.dtype == torch.bfloat16 and torch.uint8 in kept


def test_feed_forward_under_transforms_and_tangents():
    m, plain = ffn().eval(), ffn(keep8=False).eval()
    x, t = torch.randn(5, 30, 64, device=DEV), torch.randn(30, 64, device=DEV)
    assert (torch.func.vmap(m)(x) - torch.func.vmap(plain)(x)).abs().max() < 1e-5
    assert (torch.func.jacrev(lambda a: m(a).sum(0))(x[0, :3]) - torch.func.jacrev(lambda a: plain(a).sum(0))(x[0, :3])).abs().max() < 1e-5
    with fwAD.dual_level():
        got, want = (fwAD.unpack_dual(f(fwAD.make_dual(x[0], t))).tangent for f in (m, plain))
        assert (got - want).abs().max() < 1e-5
    with fwAD.dual_level():                                       # (of the second weight alone)
        tangents = []
        for f in (m, plain):
            w = f.w_2.weight.detach()
            del f.w_2.weight
            f.w_2.weight = fwAD.make_dual(w, torch.ones_like(w))
            tangents.append(fwAD.unpack_dual(f(x[0])).tangent)
        assert (tangents[0] - tangents[1]).abs().max() < 1e-4


def test_feed_forward_traced():
    m = ffn()
    x = torch.randn(30, 64, device=DEV)
    traced = torch.jit.trace(m, x)
    y = torch.randn(30, 64, device=DEV)
    assert torch.equal(traced(y), ffn(keep8=False)(y))


def test_feed_forward_of_a_subclass():
    m = ffn()
    x = torch.randn(30, 64, device=DEV)
    assert (m(x.as_subclass(Marked)).as_subclass(torch.Tensor) - ffn(keep8=False)(x)).abs().max() < 1e-5


def test_feed_forward_inside_autocast_after_a_layer_of_another_type():
    """(a first layer that answers in float32 all the same: the second one's result is the cast one's)"""
    x = torch.randn(30, 64, device=DEV)
    out = []
    for m in (ffn(), ffn(keep8=False)):
        m.w_1.register_forward_hook(lambda module, args, a: a.float())
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out.append(m(x))
    assert out[0].dtype == torch.bfloat16 and torch.equal(*out)


def test_feed_forward_with_a_transposed_weight():
    got = []
    for m in (ffn(), ffn(keep8=False)):
        m.w_2.weight = torch.nn.Parameter(m.w_2.weight.detach().t().contiguous().t())
        got.append(m(torch.ones(30, 64, device=DEV)))
    assert torch.equal(*got)
