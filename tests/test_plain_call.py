"""Which calls nothing looks into (op.plain_call), on the CPU."""
import torch
import torch.autograd.forward_ad as fwAD

from bpt_amd import op


class Marked(torch.Tensor):
    pass


def test_plain_tensors_and_arguments_left_out():
    x, w = torch.randn(3, 4), torch.nn.Parameter(torch.randn(4))
    assert op.plain_call(x) and op.plain_call(x, None, w, None)


def test_any_tensor_of_a_subclass():
    x, odd = torch.randn(3, 4), torch.randn(4).as_subclass(Marked)
    assert not op.plain_call(odd) and not op.plain_call(x, x, odd) and not op.plain_call(x, None, odd)


def test_any_tangent():
    x, w = torch.randn(3, 4), torch.randn(4)
    with fwAD.dual_level():
        assert op.plain_call(x, w)
        assert not op.plain_call(x, None, fwAD.make_dual(w, torch.ones(4))) and not op.plain_call(fwAD.make_dual(x, x), w)


def test_transforms_and_traces():
    seen = []
    f = lambda x: seen.append(op.plain_call(x)) or x * 2
    torch.func.vmap(f)(torch.randn(3, 4))
    torch.jit.trace(f, torch.randn(3), check_trace=False)
    assert seen == [False, False]
