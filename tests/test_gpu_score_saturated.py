"""Gradients of scores far beyond the cap: the derivative 1 - tanh^2(u / cap) = 1 / cosh^2 is small there, and its digits count where all scores of a row are.

Every row's |u| / cap lies within a tenth of a value between 5 and 10, so a row's derivatives differ by factors below 8 and no sum over them cancels more than
the row's ds do.  Bounds, E = 2^-24, F = half a step of bfloat16 (2^-8) or 0, as in test_gpu_score_attention, but for the derivative, which is held relatively:
exp(-2 z) with z = u / cap is off by twice z's error, the products' 72 E of sum |q k| scale / cap and 4 E |z| for the factors, 4 (e / (1 + e)) / (1 + e) by a dozen roundings."""
import math

import pytest
import torch

from test_gpu_score_attention import DEV, TYPES, close, graph, graph_args

pytestmark = pytest.mark.gpu

CAP = 2.0


def make(kind, heads, d, dtype, sign):
    src, dst, n_q, n_k = graph(kind)
    gen = torch.Generator().manual_seed(11)
    rand = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)
    way = rand(1, heads, d)
    way = way / way.norm(dim=-1, keepdim=True)
    # q.k = 8 z' cap sqrt(d / 64) along `way`, and a hundredth of it across
    rows = torch.linspace(5.0, 9.0, n_q, dtype=torch.float64)[:, None, None] * CAP * math.sqrt(d) * sign
    keys = 1 + 0.1 * torch.rand(n_k, 1, 1, generator=gen, dtype=torch.float64)
    t = TYPES[dtype]
    return dict(src=torch.from_numpy(src).long(), dst=torch.from_numpy(dst).long(), q=(rows * way / 4).to(t), k=(4 * (keys * way + 0.01 * rand(n_k, heads, d))).to(t),
                v=rand(n_k, heads, d).to(t), do=rand(n_q, heads, d).to(t))


def reference(c):
    src, dst, E = c["src"], c["dst"], 2.0 ** -24
    F = 2.0 ** -8 if c["q"].dtype == torch.bfloat16 else 0.0
    q, k, v, do = (c[n].double() for n in ("q", "k", "v", "do"))
    n_q, h, d = q.shape
    scale = 1 / math.sqrt(d)
    seg = lambda x, to, n: torch.zeros((n,) + x.shape[1:], dtype=torch.float64).index_add(0, to, x)
    qe, ke, ve, doe = q[dst], k[src], v[src], do[dst]
    u, off = (qe * ke).sum(-1) * scale, 72 * E * (qe * ke).abs().sum(-1) * scale
    z = u / CAP
    s, slope = CAP * torch.tanh(z), torch.cosh(z) ** -2
    slope_off = 2 * off / CAP + 8 * E * z.abs() + 16 * E          # relative
    assert slope_off.max() < 2e-3                                 # (first order)
    p = torch.exp(s)
    p = p / seg(p, dst, n_q)[dst]
    deg = seg(torch.ones(dst.numel(), dtype=torch.float64), dst, n_q)
    # a score is off by its products' error times the derivative, and by 12 E of itself and of lse
    rho = 2 * (off * slope + 24 * E * CAP) + (deg[dst] + 16)[:, None] * E
    o = seg(p[..., None] * ve, dst, n_q)
    o_off = seg((p * (2 * rho + F))[..., None] * ve.abs(), dst, n_q) + (deg + 16)[:, None, None] * E * seg(p[..., None] * ve.abs(), dst, n_q)
    dp, delta = (doe * ve).sum(-1), (do * o).sum(-1)
    size = (do * o).abs().sum(-1)
    delta_off = 72 * E * size + F * size + (do.abs() * o_off).sum(-1)
    ds = p * (dp - delta[dst])
    ds_off = p * (rho * (dp.abs() + delta.abs()[dst]) + 72 * E * (doe * ve).abs().sum(-1) + delta_off[dst])
    du = ds * slope * scale
    du_off = (ds_off + ds.abs() * (slope_off + F + 4 * E)) * (1 + slope_off) * slope * scale
    out = {}
    for name, to, n, y in (("dq", dst, n_q, ke), ("dk", src, k.size(0), qe)):
        g = seg(torch.ones(dst.numel(), dtype=torch.float64), to, n)
        out[name] = (seg(du[..., None] * y, to, n), seg(du_off[..., None] * y.abs(), to, n) + (g + 16)[:, None, None] * E * seg(du.abs()[..., None] * y.abs(), to, n))
    return out


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("heads,d,dtype", [(8, 64, "f32"), (16, 64, "bf16"), (6, 50, "f32"), (6, 50, "bf16"), (2, 80, "f32")])
@pytest.mark.parametrize("kind", [("window", 200, 6), ("memory", 3, 40), ("memory", 70, 5)], ids=str)
def test_scores_of_five_to_ten_caps(kind, heads, d, dtype, sign):
    from bpt_amd import op
    c = make(kind, heads, d, dtype, sign)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    q, k, v, do = (c[n].to(DEV) for n in ("q", "k", "v", "do"))
    q.requires_grad_(True), k.requires_grad_(True)
    grads = torch.autograd.grad(op.bpt_attention(*args, q, k, v, score_cap=CAP), (q, k), do)
    for (name, want), got in zip(reference(c).items(), grads):
        close(got, want, name, c["q"].dtype)


def test_the_derivative_beyond_every_exponent():
    """50 caps out cosh^2 leaves float32: 0, not NaN."""
    from bpt_amd import op
    src, dst, n, _ = graph(("window", 40, 3))
    args = graph_args(src, dst, n, n)
    for heads, d in ((8, 64), (2, 80)):
        q, k, v = (torch.full((n, heads, d), 40.0, device=DEV, requires_grad=True) for _ in range(3))
        grads = torch.autograd.grad(op.bpt_attention(*args, q, k, v, score_cap=1.0).sum(), (q, k))
        assert not any(g.any() for g in grads)
