"""Forward of few query rows with score options (the kernel that walks single rows): against the formula in 64 bits, and chosen by the call alone, whatever
calls came before it.  Tolerances of o: those of test_gpu_score_attention.  lse: off by what its scores are (12 E of their absolute values and its own, 72 E
of the products'), and by 16 E + the row's edges times E relative in the sum, all in natural units; base 2 is a factor and one rounding more."""
import math

import numpy as np
import pytest
import torch

from test_gpu_score_attention import DEV, TYPES, call, check, close, graph_args, make, on_device, reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture
def single_rows(monkeypatch):
    from bpt_amd import graphop
    monkeypatch.setattr(graphop, "SCORE_ROWS", True)


def fresh(args):
    """The same graph in tensors that no call has seen."""
    return tuple(t.clone() for t in args)


def forward(c, args):
    with torch.no_grad():
        return call(c, on_device(c, False), args, fused=True)


def log2_of_sums(c):
    """lse in base 2 and its bound."""
    D = {n: t.double() for n, t in c.items() if torch.is_tensor(t) and t.is_floating_point()}
    src, dst, (n_q, h, d), E = c["src"], c["dst"], c["q"].shape, 2.0 ** -24
    qe, ke = D["q"][dst], D["k"][src]
    u, off = (qe * ke).sum(-1) / math.sqrt(d), 72 * E * (qe * ke).abs().sum(-1) / math.sqrt(d)
    s = c["cap"] * torch.tanh(u / c["cap"]) if c["cap"] else u
    size = s.abs()
    if "slopes" in c:
        far = D["slopes"] * (D["pos_q"][dst] - D["pos_k"][src]).abs()[:, None]
        s, size = s - far, size + far
    idx = dst[:, None].expand(-1, h)
    top = torch.full((n_q, h), -1e300, dtype=torch.float64).scatter_reduce(0, idx, s, "amax")
    total = torch.zeros((n_q, h), dtype=torch.float64).index_add(0, dst, torch.exp(s - top[dst]))
    lse = torch.where(total > 0, top + torch.log(total.clamp(min=1e-300)), torch.zeros_like(top))
    worst = torch.zeros((n_q, h), dtype=torch.float64).scatter_reduce(0, idx, off + 12 * E * (size + lse[dst].abs()), "amax")
    deg = torch.zeros(n_q, dtype=torch.float64).index_add(0, dst, torch.ones(dst.numel(), dtype=torch.float64))
    return lse / math.log(2), (worst + (deg + 16)[:, None] * E) / math.log(2)


SHAPES = [(4, 64, "f32"), (8, 64, "f32"), (16, 64, "f32"), (8, 64, "bf16"), (16, 64, "bf16")]


def check_rows(kind, heads, dtype, cap, distance):
    from bpt_amd import graphop
    c = make(kind, heads, 64, dtype, cap, distance)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    want = reference(c)["o"]
    for _ in range(2):                                            # (through the plan that the first call leaves, too)
        close(forward(c, args), want, "o", TYPES[dtype])
    dev = on_device(c, False)
    score = graphop.score_options(cap or None, dev.get("slopes"), (dev["pos_q"], dev["pos_k"]) if distance else None, dev["q"], dev["k"], 0.125)
    o, lse = graphop.score_attention_forward(*args[4:], dev["q"], dev["k"], dev["v"], score, train=False)
    assert torch.equal(o, forward(c, args))
    close(lse, log2_of_sums(c), "lse", torch.float32)


# Rows of one edge, of numbers that are no multiple of four, without edges, and split ones.  Items of an (n_q, n_k) memory graph are segments of 64 edges or more,
# of the random graphs rows: 8 wavefronts an item up to 640 of them (288 of 16 heads), 4 up to 2048, beyond it 1.
@pytest.mark.parametrize("cap,distance", [(30.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("heads,d,dtype", SHAPES)
@pytest.mark.parametrize("kind", [("memory", 1, 1), ("memory", 1, 2), ("memory", 3, 67), ("memory", 1, 2048), ("memory", 2, 8191), ("random", 3, 5), ("random", 90, 1501),
                                  ("random", 1100, 4000), ("random", 4000, 9001)], ids=str)
def test_single_rows(single_rows, kind, heads, d, dtype, cap, distance):
    check_rows(kind, heads, dtype, cap, distance)


@pytest.mark.parametrize("kind,heads,dtype", [(("memory", 1, 2048), 8, "f32"), (("memory", 4, 1537), 16, "bf16"), (("memory", 8, 4096), 4, "f32")], ids=str)
def test_the_rule_takes_few_long_rows(kind, heads, dtype):
    """The call itself picks the kernel: its bits are the forced one's."""
    from bpt_amd import graphop
    c = make(kind, heads, 64, dtype, 30.0, True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c, False)
    score = graphop.score_options(30.0, dev["slopes"], (dev["pos_q"], dev["pos_k"]), dev["q"], dev["k"], 0.125)
    assert graphop._score_rows(args[6], dev["q"], 0.0, None, False)
    tiles = graphop.score_attention_forward(*args[4:], dev["q"], dev["k"], dev["v"], score, train=True)[0]
    rows = graphop.score_attention_forward(*args[4:], dev["q"], dev["k"], dev["v"], score, train=False)[0]
    assert torch.equal(forward(c, args), rows) and not torch.equal(rows, tiles)


@pytest.mark.parametrize("heads,dtype", [(8, "f32"), (16, "bf16")])
@pytest.mark.parametrize("kind", [("memory", 1, 2048), ("memory", 4, 1537)], ids=str)
def test_a_training_pass_does_not_change_a_forward_without_gradients(kind, heads, dtype):
    c = make(kind, heads, 64, dtype, 30.0, True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    first = forward(c, args)
    trained = run(c, args, True)
    assert torch.equal(forward(c, args), first)                   # forward, training, forward
    again = fresh(args)
    assert all(torch.equal(g, trained[n]) for n, g in run(c, again, True).items())
    assert torch.equal(forward(c, again), first)                  # training, forward
    run(c, again, True)
    assert torch.equal(forward(c, again), first)
