"""op.dropout: its decisions are Philox's words, its results one multiplication (and one addition) of 32 bits, rounded once."""
import numpy as np
import pytest
import torch

import philox_model
from bpt_amd import op

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SEED = 0x123456789ABCDEF


def test_known_words():
    # the generator's published vector of counter and key 0
    assert [int(w) for w in philox_model.words(0, 0, 4)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 1023, 4096, 16385, 127 * 300])
def test_elements(n, dtype):
    gen = torch.Generator().manual_seed(n)
    for p in (0.0, 0.1, 0.5, 0.999):
        for off in (0, 1):
            x, r, dy = (torch.empty(n + off, dtype=dtype, device=DEV)[off:].copy_(torch.randn(n, generator=gen)) for _ in range(3))
            kept = torch.from_numpy(philox_model.keep(SEED, p, n))
            scale = torch.tensor(1 / (1 - p), dtype=torch.float32)
            plain = lambda t: torch.where(kept, t.cpu().float() * scale, torch.zeros(()))
            leaf, other = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
            y = op.dropout(leaf, p, seed=SEED)
            (dx,) = torch.autograd.grad(y, leaf, dy)
            assert torch.equal(y.detach().cpu(), plain(x).to(dtype)) and torch.equal(dx.cpu(), plain(dy).to(dtype))
            assert torch.equal(op.dropout(x, p, seed=SEED), y)                       # (the views, and without a gradient)
            y = op.dropout(leaf, p, seed=SEED, residual=other)
            dx, dr = torch.autograd.grad(y, (leaf, other), dy)
            exact = torch.where(kept, x.cpu().double() * float(scale), torch.zeros((), dtype=torch.float64)) + r.cpu().double()
            # one rounding of the product, one of the sum, one to the type
            half = torch.finfo(dtype).eps / 2
            bound = 2 ** -24 * ((exact - r.cpu().double()).abs() + exact.abs()) + half * exact.abs()
            assert ((y.detach().cpu().double() - exact).abs() <= bound * (1 + 2 ** -7)).all()
            assert torch.equal(dx.cpu(), plain(dy).to(dtype)) and torch.equal(dr, dy)


def test_places_beyond_32_bits():
    """Elements whose counters pass 2^32 take the words that the generator has there."""
    n = 2 ** 32 + 2 ** 20 + 5
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = op.dropout(x, 0.5, seed=SEED)
    for first, count in ((2 ** 32 - 1000, 2000), (n - 1001, 1001)):
        kept = philox_model.words(SEED, first, count) >= np.uint32(2 ** 31)
        assert np.array_equal(y[first:first + count].float().cpu().numpy(), kept.astype(np.float32) * 2)
    del x, y


def test_shares_shapes_and_what_is_not_finite():
    x = torch.full((64, 1000), float("inf"), device=DEV)
    y = op.dropout(x, 0.3, seed=4)
    kept = (y != 0).float().mean().item()
    assert not y.isnan().any() and abs(kept - 0.7) < 5 * (0.21 / 64000) ** 0.5
    assert not torch.equal(y, op.dropout(x, 0.3, seed=5)) and torch.equal(y, op.dropout(x.view(-1), 0.3, seed=4).view(64, 1000))
    assert torch.equal(op.dropout(x, 0.3, seed=-1), op.dropout(x, 0.3, seed=2 ** 64 - 1))
    assert op.dropout(torch.empty(0, 5, device=DEV), 0.5).shape == (0, 5) and op.dropout(torch.tensor(2.0, device=DEV), 0.0) == 2
    # the highest seed word matters
    assert not torch.equal(y, op.dropout(x, 0.3, seed=4 + 2 ** 32))


def test_twice_differentiable():
    x = torch.randn(40, device=DEV, requires_grad=True)
    y = op.dropout(x * x, 0.4, seed=8)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    (ddx,) = torch.autograd.grad(dx.sum(), x)
    assert torch.equal(ddx.cpu(), torch.where(torch.from_numpy(philox_model.keep(8, 0.4, 40)), torch.tensor(1 / (1 - 0.4), dtype=torch.float32) * 2, torch.zeros(())))


def test_captured():
    x = torch.randn(3000, device=DEV)
    graph = torch.cuda.CUDAGraph()
    op.dropout(x, 0.2, seed=6)
    with torch.cuda.graph(graph):
        y = op.dropout(x, 0.2, seed=6)
    for turn in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, op.dropout(x, 0.2, seed=6))


def test_refusals():
    x = torch.randn(4, 8, device=DEV)
    for exc, call in [(ValueError, lambda: op.dropout(x, 1.0)), (ValueError, lambda: op.dropout(x, -0.5)), (ValueError, lambda: op.dropout(x, 0.1, residual=x[:2])),
                      (RuntimeError, lambda: op.dropout(x.t(), 0.1)), (RuntimeError, lambda: op.dropout(x.double(), 0.1)), (RuntimeError, lambda: op.dropout(x.cpu(), 0.1)),
                      (RuntimeError, lambda: op.dropout(x, 0.1, residual=x.bfloat16()))]:
        with pytest.raises(exc):
            call()
