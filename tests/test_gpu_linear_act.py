"""op.linear_act against its formula in 64 bits: every form of the products, epilogues, gradients, odd sizes and places, streams, captures.

Bounds, u = 2^-24, v half a step of the type (2^-24, 2^-8): a is off by (inner + 8) u S, S = |x| |w|^T + |b| (each product and each addition rounds once; products of
bfloat16 are exact); an activation passes that on by at most 1.13 (gelu's steepest) and adds 16 u of its own for erfc and its product; dropout and the
residual round once each; the result rounds by v.  g = dy keep act'(a) is off by v |g|, and by 0.8 |dy keep| times what a is off by where gelu (0.8: its second
derivative), of which v |a| is the kept tensor's rounding, and 16 u; where relu and a within its error of 0, by |dy keep|.  A product of g is off by
what g is off by, summed with the other factor's absolute values, by (terms + 8) u of the sum of absolute products, and by v of itself."""
import math

import numpy as np
import pytest
import torch

from bpt_amd import op
from philox_model import keep

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def inputs(rows, inner, outer, dtype, bias, residual, seed=0, off=0):
    gen = torch.Generator().manual_seed(seed + 7 * rows + 3 * inner + outer)

    def make(*shape, scale=1.0):
        n = math.prod(shape)
        buf = torch.empty(n + off, dtype=dtype, device=DEV)
        t = buf[off:].view(shape)                       # (off: a start that lies on no 16 bytes)
        return t.copy_((torch.randn(n, generator=gen) * scale).view(shape))
    return dict(x=make(rows, inner), w=make(outer, inner, scale=inner ** -0.5), b=make(outer, scale=0.3) if bias else None,
                r=make(rows, outer) if residual else None, dy=make(rows, outer, scale=0.125))


def expected(t, act, p, seed):
    """{name: (value, bound)} of the result and the gradients, in 64 bits."""
    d = {n: None if v is None else v.detach().double() for n, v in t.items()}
    v = HALF[t["x"].dtype]
    (rows, inner), outer = d["x"].shape, d["w"].size(0)
    a, s = d["x"] @ d["w"].T, d["x"].abs() @ d["w"].abs().T
    if d["b"] is not None:
        a, s = a + d["b"], s + d["b"].abs()
    ea = (inner + 8) * U * s
    cdf = torch.special.ndtr(a)
    y, ey = a, ea
    if act == "relu":
        y = a.clamp(min=0)
    elif act == "gelu":
        y, ey = a * cdf, 1.13 * ea + 16 * U * a.abs()
    scale = torch.ones_like(a)
    if p:
        scale = torch.from_numpy(keep(seed, p, rows * outer)).to(DEV).view(rows, outer).double() / (1 - p)
        y, ey = y * scale, ey * scale + 2 * U * (y * scale).abs()
    if d["r"] is not None:
        y = y + d["r"]
        ey = ey + U * (y.abs() + d["r"].abs())
    out = {"y": (y, ey + v * y.abs() + v * ey)}
    h = d["dy"] * scale
    g, eg = h, 2 * U * h.abs()
    if act == "relu":
        g = h * (a > 0)
        eg = eg + h.abs() * (a.abs() <= ea)
    elif act == "gelu":
        g = h * (cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi))
        eg = eg + h.abs() * (0.8 * (ea + v * a.abs()) + 16 * U)
    sums = eg + (rows + 8) * U * g.abs()                # (the bias gradient's terms are not rounded to the type first)
    if act or p:
        eg = eg + v * g.abs()
    product = lambda l, el, r_, n: (l @ r_, el @ r_.abs() + (n + 8) * U * (l.abs() @ r_.abs()) + v * (l @ r_).abs())
    out["dx"] = product(g, eg, d["w"], outer)
    out["dw"] = product(g.T, eg.T, d["x"], rows)
    if d["b"] is not None:
        out["db"] = (g.sum(0), sums.sum(0) + v * g.sum(0).abs())
    return out


def check(got, want, what):
    value, bound = want
    err = (got.double() - value).abs()
    worst = (err / (bound + 1e-30)).max().item() if err.numel() else 0.0
    assert got.isfinite().all() and worst <= 1.0, f"{what}: {worst} times the bound"


def run(t, act, p, seed):
    leaves = {n: v.detach().requires_grad_(True) for n, v in t.items() if v is not None and n != "dy"}
    y = op.linear_act(leaves["x"], leaves["w"], leaves.get("b"), activation=act, residual=leaves.get("r"), dropout_p=p, seed=seed)
    grads = torch.autograd.grad(y, list(leaves.values()), t["dy"])
    return dict(zip(("d" + n for n in leaves), grads), y=y.detach())


SIZES = [(1, 1, 1), (1, 512, 2048), (3, 7, 5), (16, 64, 64), (17, 33, 66), (48, 512, 512), (64, 65, 16), (65, 128, 64), (130, 300, 129), (257, 301, 255), (300, 8, 1000),
         (640, 1040, 136), (2000, 256, 512), (4099, 64, 520), (66, 4096, 72), (32, 1024, 200), (33, 2049, 130), (64, 2050, 66), (17, 5000, 40)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_products_and_epilogues(size, dtype):
    for i, (act, bias, residual, p) in enumerate([(None, False, False, 0.0), ("relu", True, False, 0.1), ("gelu", True, True, 0.0), ("relu", False, True, 0.3),
                                                  (None, True, True, 0.5)]):
        t = inputs(*size, dtype, bias, residual, seed=i)
        got, want = run(t, act, p, 12345678901234567 + i), expected(t, act, p, 12345678901234567 + i)
        for name, w in want.items():
            check(got[name], w, f"{size} {act} bias={bias} residual={residual} p={p} {name}")
        if residual:
            assert torch.equal(got["dr"], t["dy"])
        again = run(t, act, p, 12345678901234567 + i)
        assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [9, 200])
def test_tensors_that_start_anywhere(rows, dtype):
    for off in (1, 2, 3):
        t = inputs(rows, 96, 100, dtype, True, True, off=off)
        got, want = run(t, "gelu", 0.2, 5), expected(t, "gelu", 0.2, 5)
        for name, w in want.items():
            check(got[name], w, f"off={off} {name}")


@pytest.mark.parametrize("rows", [40, 300])
def test_what_is_not_finite_stays_in_its_row(rows):
    t = inputs(rows, 200, 72, torch.float32, True, False)
    t["x"][rows - 1] = float("inf")
    t["x"][3, 17] = float("nan")
    y = op.linear_act(t["x"], t["w"], t["b"], activation="relu")
    odd = ~y.isfinite().all(1)
    assert odd[3] and odd[rows - 1] and odd.sum() == 2 and y[3].isnan().all()
    # a dropped infinity is 0
    z = op.linear_act(t["x"][rows - 1:].clamp(max=3e38), t["w"].abs(), activation=None, dropout_p=0.5, seed=1)
    assert (z == 0).any() and not z.isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(8190, 1100, 1540), (8190, 1540, 1100), (33001, 1500, 1500), (4099, 300, 302), (5000, 2050, 130)], ids=str)
def test_large_tiles_and_ragged_reductions(size, dtype):
    t = inputs(*size, dtype, True, False, seed=9)
    got, want = run(t, "relu", 0.1, 77), expected(t, "relu", 0.1, 77)
    for name, w in want.items():
        check(got[name], w, f"{size} {name}")


@pytest.mark.parametrize("size", [(40, 256, 72), (300, 256, 200), (1300, 1100, 1540)], ids=str)
@pytest.mark.parametrize("x_by,w_by", [(2.0 ** -120, 2.0 ** 10), (2.0 ** -115, 2.0 ** 15), (2.0 ** -100, 1.0), (2.0 ** 100, 2.0 ** -20), (2.0 ** 124, 2.0 ** -60)])
def test_low_and_high_numbers(size, x_by, w_by):
    """Products of numbers near either end of float32's range are as exact as others, where no sum of their terms can leave it, in whatever order they are added: where the terms'
    absolute values together lie within it.  (Hundreds of terms of dw with x of 2^124 do not: 0.1 2^124 300 is 2^129.)"""
    t = inputs(*size, torch.float32, False, False, seed=2)
    t["x"], t["w"] = t["x"].clamp(-2, 2) * x_by, t["w"] * w_by
    got, want = run(t, None, 0.0, 0), expected(t, None, 0.0, 0)
    x, w, dy = (t[n].double().abs() for n in ("x", "w", "dy"))
    for name, terms in (("y", x @ w.T), ("dw", dy.T @ x)):
        if terms.max() <= torch.finfo(torch.float32).max:
            check(got[name], want[name], f"{size} {x_by} {name}")
        else:
            assert name == "dw" and x_by == 2.0 ** 124


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(300, 300, 302), (130, 44, 68), (700, 1030, 258)], ids=str)
def test_what_stands_behind_a_row_does_not_reach_it(size, dtype):
    """Rows of NaN next to those that count, and behind the tensors' ends."""
    rows, inner, outer = size
    t = inputs(*size, dtype, False, False, seed=3)
    odd = {n: torch.full((v.size(0) + 100, v.size(1)), float("nan"), dtype=dtype, device=DEV) for n, v in t.items() if n in ("x", "w", "dy")}
    for n, whole in odd.items():
        whole[:t[n].size(0)] = t[n]
    there = dict(t, **{n: whole[:t[n].size(0)] for n, whole in odd.items()})
    a, b = run(t, None, 0.0, 0), run(there, None, 0.0, 0)
    assert all(torch.equal(a[n], b[n]) for n in a)
    t["x"][5], t["w"][7] = float("nan"), float("nan")
    y = op.linear_act(t["x"], t["w"])
    assert y[5].isnan().all() and y[:, 7].isnan().all()
    y[5], y[:, 7] = 0, 0
    assert y.isfinite().all()


def test_leading_axes_nothing_and_one_gradient():
    t = inputs(24, 40, 12, torch.float32, True, True)
    flat = run(t, "gelu", 0.1, 3)
    shaped = {n: v if n in "wb" else v.view(2, 3, 4, -1) for n, v in t.items()}
    got = run(shaped, "gelu", 0.1, 3)
    assert got["y"].shape == (2, 3, 4, 12) and all(torch.equal(got[n].reshape(flat[n].shape), flat[n]) for n in flat)
    for shape in ((0, 40), (2, 0, 40)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        w, b = t["w"].detach().requires_grad_(True), t["b"].detach().requires_grad_(True)
        y = op.linear_act(x, w, b, activation="relu", dropout_p=0.1)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert y.shape == shape[:-1] + (12,) and dx.shape == x.shape and not dw.any() and not db.any()
    x = t["x"].detach().requires_grad_(True)
    y = op.linear_act(x, torch.empty(0, 40, device=DEV), torch.empty(0, device=DEV))
    assert y.shape == (24, 0) and not torch.autograd.grad(y, x, torch.zeros_like(y))[0].any()
    y = op.linear_act(t["x"][0], t["w"], t["b"])                  # one row without an axis of rows
    assert torch.equal(y, op.linear_act(t["x"][:1], t["w"], t["b"])[0])
    for only in "xwbr":                                            # any one of the gradients alone
        leaves = {n: v.detach().requires_grad_(n == only) for n, v in t.items()}
        y = op.linear_act(leaves["x"], leaves["w"], leaves["b"], activation="gelu", residual=leaves["r"], dropout_p=0.1, seed=3)
        (grad,) = torch.autograd.grad(y, leaves[only], t["dy"])
        assert torch.equal(grad, flat["d" + only])


def test_gradients_are_differences():
    """The formula's gradients against central differences of the formula's results, in the kernels' own 32 bits: h = 2^-6 leaves h^2 / 6 of a third derivative (gelu's is
    below 1.6, and so is any product of three of x's and w's entries here) and 4 u |sum| / h of rounding."""
    t = inputs(5, 6, 7, torch.float32, True, True)
    got = run(t, "gelu", 0.25, 11)
    h = 2.0 ** -6
    for name in ("x", "w", "b", "r"):
        flat = t[name].view(-1)
        for i in range(0, flat.numel(), 5):
            both = []
            for sign in (1, -1):
                moved = {n: v.clone() if v is not None else None for n, v in t.items()}
                moved[name].view(-1)[i] += sign * h
                y = op.linear_act(moved["x"], moved["w"], moved["b"], activation="gelu", residual=moved["r"], dropout_p=0.25, seed=11)
                both.append((y.double() * t["dy"].double()).sum())
            assert abs((both[0] - both[1]) / (2 * h) - got["d" + name].view(-1)[i].double()) < 1e-3


def test_another_stream_and_a_captured_step():
    t = inputs(700, 256, 320, torch.bfloat16, True, True)
    want = run(t, "relu", 0.1, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, "relu", 0.1, 9)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(t, "relu", 0.1, 9)
    for turn in range(3):
        t["x"].copy_(inputs(700, 256, 320, torch.bfloat16, True, True, seed=turn)["x"])
        graph.replay()
        torch.cuda.synchronize()
        want = run(t, "relu", 0.1, 9)
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_long_rows_of_many_bytes():
    """A result of more than 2^32 bytes: the last rows are what they are alone."""
    rows, inner, outer = 540000, 16, 2048
    x = torch.randn(rows, inner, device=DEV)
    w = torch.randn(outer, inner, device=DEV)
    y = op.linear_act(x, w, activation="relu", dropout_p=0.0)
    assert y.numel() * 4 > 2 ** 32
    tail = op.linear_act(x[-300:].contiguous(), w, activation="relu")
    assert torch.equal(y[-300:], tail)
    del y


def test_more_columns_than_a_launch_of_few_rows_has_threads_for():
    outer = 2 ** 27 + 5
    x, w = torch.full((1, 1), 3.0, device=DEV), torch.arange(outer, dtype=torch.float32, device=DEV).view(-1, 1)
    assert torch.equal(op.linear_act(x, w).view(-1), 3.0 * w.view(-1))


def test_seeds_come_from_torch():
    t = inputs(20, 32, 64, torch.float32, False, False)
    torch.manual_seed(5)
    a = op.linear_act(t["x"], t["w"], dropout_p=0.5)
    b = op.linear_act(t["x"], t["w"], dropout_p=0.5)
    torch.manual_seed(5)
    assert torch.equal(a, op.linear_act(t["x"], t["w"], dropout_p=0.5)) and not torch.equal(a, b)


def test_refusals():
    x, w = torch.randn(4, 8, device=DEV), torch.randn(6, 8, device=DEV)
    for exc, call in [
            (ValueError, lambda: op.linear_act(x, w, activation="tanh")), (ValueError, lambda: op.linear_act(x, w, dropout_p=1.0)),
            (ValueError, lambda: op.linear_act(x, w, dropout_p=-0.1)), (ValueError, lambda: op.linear_act(x, w, dropout_p=float("nan"))),
            (ValueError, lambda: op.linear_act(x, w.t().contiguous())), (ValueError, lambda: op.linear_act(x, w, torch.randn(5, device=DEV))),
            (ValueError, lambda: op.linear_act(x, w, residual=x)), (RuntimeError, lambda: op.linear_act(x, w.bfloat16())),
            (RuntimeError, lambda: op.linear_act(x.double(), w.double())), (RuntimeError, lambda: op.linear_act(x.half(), w.half())),
            (RuntimeError, lambda: op.linear_act(x.t(), w)), (RuntimeError, lambda: op.linear_act(x, w.cpu())),
            (RuntimeError, lambda: op.linear_act(x, w[:, ::2])), (ValueError, lambda: op.linear_act(x[:, :0].contiguous(), w[:, :0].contiguous()))]:
        with pytest.raises(exc):
            call()
    x.requires_grad_(True)
    y = op.linear_act(x, w, activation="gelu")
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
