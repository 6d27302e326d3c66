"""Rows whose every score lies far below zero, as slopes times distances of 10^10 are: softmax does not change when a row's scores move together, so the
nearest key is all there is.  The distances of a row differ by 10^10 (slopes of 1), the products are a few units: p is exactly 1 and 0, o and dv are
exact copies and sums, dq and dk zero times finite numbers, and the slopes' gradient, zero too, is off by the row's ds times the distance: ds by 2 * 72
roundings of sum |dO v| (and, in bfloat16, o is v as it is)."""
import pytest
import torch

from test_gpu_score_attention import DEV, TYPES, graph_args

pytestmark = pytest.mark.gpu

APART = 2.0 ** 34


def make(n_q, n_k, heads, d, dtype):
    gen = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=gen).to(TYPES[dtype]).to(DEV)
    order = torch.randperm(n_k, generator=gen)
    pos_k = (1 + order.float()) * APART                           # key `nearest` is one step away from every query, the next one two
    src, dst = torch.arange(n_k).repeat(n_q), torch.arange(n_q).repeat_interleave(n_k)
    return (graph_args(src.numpy(), dst.numpy(), n_q, n_k), rand(n_q, heads, d), rand(n_k, heads, d), rand(n_k, heads, d), rand(n_q, heads, d),
            torch.zeros(n_q, device=DEV), pos_k.to(DEV), int(order.argmin()))


SHAPES = [(8, 64, "f32"), (4, 64, "f32"), (16, 64, "bf16"), (8, 64, "bf16"), (6, 50, "f32"), (6, 50, "bf16"), (2, 80, "f32"), (8, 64, "f64")]


@pytest.mark.parametrize("cap", [None, 10.0])
@pytest.mark.parametrize("heads,d,dtype", SHAPES)
@pytest.mark.parametrize("n_q,n_k", [(1, 1), (40, 6), (5, 700), (1, 4100), (300, 40)])
def test_the_nearest_key_is_taken(n_q, n_k, heads, d, dtype, cap):
    """Whole rows, rows split over segments, tiles in parts, and (without gradients) rows walked one by one."""
    from bpt_amd import op
    args, q, k, v, do, pos_q, pos_k, nearest = make(n_q, n_k, heads, d, dtype)
    slopes = torch.ones(heads, device=DEV)
    want = v[nearest].expand(n_q, heads, d)
    with torch.no_grad():
        assert torch.equal(op.bpt_attention(*args, q, k, v, score_cap=cap, slopes=slopes, pos=(pos_q, pos_k)), want)
    leaves = [x.requires_grad_(True) for x in (q, k, v, slopes)]
    o = op.bpt_attention(*args, q, k, v, score_cap=cap, slopes=slopes, pos=(pos_q, pos_k))
    dq, dk, dv, dslopes = torch.autograd.grad(o, leaves, do)
    assert torch.equal(o, want)
    total = do.double().sum(0)
    off = (n_q + 1) * 2.0 ** -24 * do.double().abs().sum(0) + torch.finfo(TYPES[dtype]).eps / 2 * total.abs()
    assert ((dv[nearest].double() - total).abs() <= off).all()
    dv[nearest] = 0
    assert not dv.any()
    size = (do.double() * want.double()).abs().sum(-1)            # (n_q, heads)
    ds = 2 * 72 * 2.0 ** -24 * size
    scale = d ** -0.5
    rounded = torch.finfo(TYPES[dtype]).eps
    assert (dq.double().abs() <= (ds[..., None] * scale * k[nearest].double().abs()) * (1 + 2 * rounded)).all()
    assert (dk.double().abs() <= (ds[..., None] * scale * q.double().abs()).sum(0) * (1 + 2 * rounded)).all()
    assert (dslopes.double().abs() <= ds.sum(0) * APART * (1 + 1e-6)).all()


def test_single_rows(monkeypatch):
    from bpt_amd import graphop, op
    monkeypatch.setattr(graphop, "SCORE_ROWS", True)
    for heads, dtype in ((8, "f32"), (16, "bf16")):
        for n_q, n_k in ((1, 1), (1, 4100), (700, 3), (2500, 2)):
            args, q, k, v, _, pos_q, pos_k, nearest = make(n_q, n_k, heads, 64, dtype)
            with torch.no_grad():
                o = op.bpt_attention(*args, q, k, v, slopes=torch.ones(heads, device=DEV), pos=(pos_q, pos_k))
            assert torch.equal(o, v[nearest].expand_as(o)), (heads, dtype, n_q, n_k)


@pytest.mark.parametrize("heads,d,dtype", [(8, 64, "f32"), (6, 50, "bf16"), (2, 80, "f32")])
def test_rows_without_edges_stay_empty(heads, d, dtype):
    from bpt_amd import op
    src, dst = torch.tensor([0, 1, 2]), torch.tensor([1, 1, 4])
    args = graph_args(src.numpy(), dst.numpy(), 6, 6)
    q, k, v = (torch.randn(6, heads, d, device=DEV).to(TYPES[dtype]).requires_grad_(True) for _ in range(3))
    pos = torch.tensor([3.0, 1.0, 2.0, 0.0, -2.0, 5.0], device=DEV) * APART
    o = op.bpt_attention(*args, q, k, v, slopes=torch.ones(heads, device=DEV), pos=pos)
    assert torch.equal(o[1], v[1]) and torch.equal(o[4], v[2])      # (row 1 is its own neighbour and that of row 0, two steps away)
    assert not o[[0, 2, 3, 5]].any()
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
    assert not dq[[0, 2, 3, 5]].any() and not dk[[0, 3, 4, 5]].any() and torch.equal(dv[2], torch.ones_like(dv[2])) and not dv[0].any()
