"""op.linear_act's float32 products over the whole range of float32, in each of the three products of a layer, and how exact one product is.

Bounds, u = 2^-24: a sum of n products is off by (n + 8) u of the sum of their absolute values, as in the tests of ordinary numbers.  Below float32's normal numbers a rounding
is off by half of its lowest number, 2^-150, whatever the value: one for each product that the float32 instructions form, one for each share of a reduction elsewhere, and sums of such
multiples are exact, so n 2^-150 together."""
import pytest
import torch

from bpt_amd import op

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
SIZES = [(40, 256, 72), (300, 256, 200), (257, 301, 255), (1300, 1100, 1540), (8190, 1100, 1540)]      # few rows; tiles of 64, of 64 through registers, of 128, of 256


def inputs(size, by):
    rows, inner, outer = size
    gen = torch.Generator().manual_seed(rows)
    shapes = dict(x=(rows, inner), w=(outer, inner), dy=(rows, outer))
    return {n: (torch.randn(shape, generator=gen).clamp(-2, 2) * s).to(DEV) for (n, shape), s in zip(shapes.items(), by)}


def results(t):
    x, w = t["x"].detach().requires_grad_(True), t["w"].detach().requires_grad_(True)
    y = op.linear_act(x, w)
    return (y.detach(), *torch.autograd.grad(y, (x, w), t["dy"]))


def compare(name, got, a, b):
    a, b = a.double(), b.double()
    want, terms = a @ b, a.abs() @ b.abs()
    assert terms.max() < torch.finfo(torch.float32).max
    worst = ((got.double() - want).abs() / ((a.size(1) + 8) * U * terms + a.size(1) * 2.0 ** -150)).max().item()
    assert worst <= 1.0, f"{name}: {worst} times the bound"


def check(t):
    y, dx, dw = results(t)
    compare("y", y, t["x"], t["w"].T)
    compare("dx", dx, t["dy"], t["w"])
    compare("dw", dw, t["dy"].T, t["x"])


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("x,w,dy", [(-123, 40, -123), (-118, 60, -118), (60, -118, 20), (-126, 100, -126), (-130, 60, -130), (40, -140, 40), (-130, 100, -110), (-105, 20, 0),
                                    (-100, 0, -145), (-70, -70, 0)])
def test_low_numbers_times_high_ones(size, x, w, dy):
    """Operands whose lower digits, or all of them, lie below float32's normal numbers, times others that bring them back into its middle."""
    check(inputs(size, (2.0 ** x, 2.0 ** w, 2.0 ** dy)))


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_low_numbers_beside_ordinary_ones(size):
    """Some columns low in x and high in the weight, the others ordinary: what the low ones add is as large as what those do.  (dx's high columns can leave float32's range.)"""
    t = inputs(size, (1.0, 1.0, 1.0))
    t["x"][:, ::3] *= 2.0 ** -127
    t["w"][:, ::3] *= 2.0 ** 125
    y, dx, dw = results(t)
    others = torch.arange(size[1], device=DEV) % 3 != 0
    compare("y", y, t["x"], t["w"].T)
    compare("dx", dx[:, others], t["dy"], t["w"][:, others])
    compare("dw", dw, t["dy"].T, t["x"])


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_low_numbers_beside_what_is_not_finite(size):
    t = inputs(size, (2.0 ** -123, 2.0 ** 40, 2.0 ** -123))
    t["x"][5], t["dy"][5] = float("inf"), float("nan")
    y, dx, _ = results(t)
    assert not y[5].isfinite().any() and dx[5].isnan().all()
    others = torch.arange(size[0], device=DEV) != 5
    compare("y", y[others], t["x"][others], t["w"].T)
    compare("dx", dx[others], t["dy"][others], t["w"])


@pytest.mark.parametrize("size", [(65, 33), (300, 200), (4096, 4096)], ids=str)
def test_a_product_of_two_numbers(size):
    """x w of two numbers, by tiles: what the products of bfloat16 leave out is below 2^-21 (1 + 2^-9) = 8.02 u of it and makes it smaller; adding up its parts is off by
    a step of 2 u at most where the last and largest is added, by 2^-6 of one at each of three before."""
    rows, outer = size
    gen = torch.Generator().manual_seed(outer)
    any_number = lambda n: (torch.randint(0, 2 ** 23, (n,), generator=gen, dtype=torch.int32) + 0x3F800000).view(torch.float32)
    x, w = torch.zeros(rows, 96, device=DEV), torch.zeros(outer, 96, device=DEV)
    x[:, 40], w[:, 40] = any_number(rows).to(DEV), any_number(outer).to(DEV)
    x[3, 40] = w[5, 40] = 1 + 2.0 ** -7 - 2.0 ** -23                # (the lower thirds of either as large as they get)
    want = x[:, 40, None].double() * w[None, :, 40].double()
    off = (op.linear_act(x, w).double() - want) / (U * want)
    assert off.min() >= -(8.02 + 2 + 0.1) and off.max() <= 2 + 0.1
