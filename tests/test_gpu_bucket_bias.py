"""op.bpt_attention with a bias by buckets (bias_table, buckets) and op.bucket_bias against the formula in 64 bits.

Tolerances, from the arithmetic, per element.  E = 2^-24; F = half a step of the result's type beyond float32 (bfloat16 2^-8, else 0).
  score  s = scale q.k + table: 64 products and their sum, 72 E of the sum of absolute values; the table's value three roundings of its own, the sums and the difference
         to lse: 12 E of the absolute values of what is added, with lse
  p      relative: exp2 of that once for the pair and once for the row's sum, and (edges of the row + 16) E for the sum
  o      the relative error of p twice over sum p |v|, (edges + 16) E of it, F for p rounded on its way into the product
  dp, delta   72 E of the sums of absolute values; delta uses o as stored (F of sum |dO| |o| more)
  ds     the relative error of p (|dp| + |delta|), those two errors times p; scaled and unscaled again 4 E; F for ds rounded on its way into dq and dk
  dq, dk, dv  sums of such terms over edges: their bounds' sums and (edges + 16) E of the sum of absolute values
  dtable      the same over the edges of a bucket; no sum there has more than edges / 4096 + 600 terms in turn, so (edges / 4096 + 600) E of the sum of absolute values
and half a step of the result's type.  The chain of operators stores tensors of an edge's size between them, each of which rounds F once more: q.k (F |scale q.k| of a score), dL/dp
(p F (|dp| + sum p |dp|) of ds) and ds on its way to the table (F |ds|)."""
import math

import numpy as np
import pytest
import torch

from test_gpu_score_attention import TYPES, close, graph, graph_args, make as make_scores

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(kind, heads, d, dtype, n=20, cap=0.0, distance=False, seed=0):
    c = make_scores(kind, heads, d, dtype, cap, distance, seed=seed)
    gen = np.random.default_rng(seed + 9)
    c["bias_table"] = torch.from_numpy(gen.normal(size=(n, heads)) * 0.7).to(TYPES[dtype])
    # (a few edges without a bucket, as -1, n and far beyond)
    b = gen.integers(0, n, c["src"].numel())
    for i, odd in enumerate((-1, n, 2 ** 40, -2 ** 63)):
        b[i * 7 + 3::97] = odd
    c["buckets"] = torch.from_numpy(b)
    return c


def reference(c, drop=None, chain=False):
    """{name: (value, bound)} in 64 bits."""
    src, dst, buckets = c["src"], c["dst"], c["buckets"]
    D = {n: t.double() for n, t in c.items() if torch.is_tensor(t) and t.is_floating_point()}
    q, k, v, do = (D[n] for n in ("q", "k", "v", "do"))
    n_q, h, d = q.shape
    n_b = D["bias_table"].size(0)
    n_e, scale, cap, E = src.numel(), 1 / math.sqrt(d), c["cap"], 2.0 ** -24
    F = 2.0 ** -8 if c["q"].dtype == torch.bfloat16 else 0.0
    seg = lambda x, to, n: torch.zeros((n,) + x.shape[1:], dtype=torch.float64).index_add(0, to, x)
    qe, ke, ve, doe = q[dst], k[src], v[src], do[dst]
    there = (buckets >= 0) & (buckets < n_b)
    bias = torch.where(there[:, None], D["bias_table"][torch.where(there, buckets, 0)], 0.0)
    ax = (qe * ke).abs().sum(-1)
    u = (qe * ke).sum(-1) * scale + bias
    hidden = u == -math.inf
    finite = torch.where(hidden, 0.0, u)
    du_err = 72 * E * ax * scale + 3 * E * torch.where(hidden, 0.0, bias).abs()
    if chain:
        du_err = du_err + F * (qe * ke).sum(-1).abs() * scale
    t = torch.tanh(u / cap) if cap else None
    s = cap * t if cap else torch.where(hidden, -math.inf, u)
    slope = 1 - t * t if cap else torch.ones_like(u)
    mag = finite.abs() + torch.where(hidden, 0.0, bias).abs()
    if "slopes" in c:
        far = (D["pos_q"][dst] - D["pos_k"][src]).abs()[:, None]
        s = s - D["slopes"] * far
        mag = mag + D["slopes"] * far
    idx = dst[:, None].expand(-1, h)
    top = torch.full((n_q, h), -1e300, dtype=torch.float64).scatter_reduce(0, idx, s, "amax")
    w = torch.where(hidden, 0.0, torch.exp(torch.where(hidden, 0.0, s - top[dst])))
    total = seg(w, dst, n_q)
    p = torch.where(total[dst] > 0, w / total[dst], 0.0)
    lse = torch.where(total > 0, torch.log(total.clamp(min=1e-300)) + top, 0.0)
    err_s = du_err + 12 * E * (mag + lse[dst].abs())
    deg = torch.zeros(n_q, dtype=torch.float64).index_add(0, dst, torch.ones(n_e, dtype=torch.float64))
    row_err = torch.zeros((n_q, h), dtype=torch.float64).scatter_reduce(0, idx, err_s, "amax")
    rho = err_s + row_err[dst] + (deg[dst] + 16)[:, None] * E
    m = drop if drop is not None else torch.ones_like(p)
    o = seg((p * m)[..., None] * ve, dst, n_q)
    o_b = seg((p * m * (2 * rho + F))[..., None] * ve.abs(), dst, n_q) + (deg + 16)[:, None, None] * E * seg((p * m)[..., None] * ve.abs(), dst, n_q)
    dp, adp = (doe * ve).sum(-1), (doe * ve).abs().sum(-1)
    delta, adelta = (do * o).sum(-1), (do * o).abs().sum(-1)
    delta_b = 72 * E * adelta + F * adelta + (do.abs() * o_b).sum(-1)
    ds = p * (dp * m - delta[dst])
    ds_b = p * (rho * (dp.abs() * m + delta.abs()[dst]) + 72 * E * adp * m + delta_b[dst])
    if chain:
        ds_b = ds_b + p * F * (dp.abs() * m + seg(p * m * dp.abs(), dst, n_q)[dst])
    dx, dx_b = ds * slope, ds_b * slope + ds.abs() * 8 * E + 4 * E * (ds * slope).abs()
    du, du_b = dx * scale, (dx_b + F * dx.abs()) * scale
    out = {"o": (o, o_b)}
    deg_k = torch.zeros(k.size(0), dtype=torch.float64).index_add(0, src, torch.ones(n_e, dtype=torch.float64))
    pm, pm_b = p * m, p * m * (rho + F)
    for name, to, n, g, a, a_b, y in (("dq", dst, n_q, deg, du, du_b, ke), ("dk", src, k.size(0), deg_k, du, du_b, qe), ("dv", src, k.size(0), deg_k, pm, pm_b, doe)):
        out[name] = (seg(a[..., None] * y, to, n), seg(a_b[..., None] * y.abs(), to, n) + (g + 16)[:, None, None] * E * seg(a.abs()[..., None] * y.abs(), to, n))
    rows = torch.where(there, buckets, n_b)
    out["dbias_table"] = (seg(dx, rows, n_b + 1)[:n_b], (seg(dx_b, rows, n_b + 1) + (n_e / 4096 + 600) * E * seg(dx.abs(), rows, n_b + 1))[:n_b])
    if chain:
        out["dbias_table"] = (out["dbias_table"][0], out["dbias_table"][1] + F * seg(dx.abs(), rows, n_b + 1)[:n_b])
    if "slopes" in c:
        out["dslopes"] = (-(ds * far).sum(0), (ds_b * far).sum(0) + (n_e / 16 + 64) * E * (ds * far).abs().sum(0))
    return out


def call(c, dev, args, fused=None, **kw):
    from bpt_amd import op
    opts = dict(bias_table=dev["bias_table"], buckets=dev["buckets"])
    if c["cap"]:
        opts["score_cap"] = c["cap"]
    if "slopes" in c:
        opts.update(slopes=dev["slopes"], pos=dev["pos_q"] if c["pos_q"] is c["pos_k"] else (dev["pos_q"], dev["pos_k"]))
    return op.bpt_attention(*args, dev["q"], dev["k"], dev["v"], fused=fused, **opts, **kw)


LEAVES = ("q", "k", "v", "slopes", "bias_table")


def on_device(c, grad=True):
    return {n: t.to(DEV).requires_grad_(grad and n in LEAVES) for n, t in c.items() if torch.is_tensor(t)}


def run(c, args, fused=None, **kw):
    dev = on_device(c)
    o = call(c, dev, args, fused, **kw)
    names = [n for n in LEAVES if n in dev]
    return dict({"o": o.detach()}, **{"d" + n: g for n, g in zip(names, torch.autograd.grad(o, [dev[n] for n in names], dev["do"]))})


def check(c, fused=None, drop=None, **kw):
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    ref = reference(c, drop, chain=fused is False)
    first = None
    for _ in range(2):
        got = run(c, args, fused, **kw)
        for n, want in ref.items():
            close(got[n], want, n, torch.float32 if n == "dslopes" else c["q"].dtype)
        assert first is None or all(torch.equal(first[n], got[n]) for n in got)
        first = got
    with torch.no_grad():
        dev = on_device(c, False)
        close(call(c, dev, args, fused, **kw), ref["o"], "o without gradients", c["q"].dtype)
        if fused:                                                 # (nor without the side that only a backward reads)
            close(call(c, dev, (None,) * 4 + tuple(args[4:]), fused, **kw), ref["o"], "o of one side", c["q"].dtype)
    return args, got


GRAPHS = [("bpt", 1, 1), ("bpt", 5, 2), ("bpt", 33, 4), ("bpt", 700, 4), ("window", 300, 20), ("random", 90, 1500), ("random", 3, 5), ("random", 1000, 300),
          ("memory", 1, 700), ("memory", 17, 3), ("memory", 1, 1), ("memory", 40, 300)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", GRAPHS, ids=str)
def test_matches_the_formula(kind, dtype):
    check(make(kind, 8, 64, dtype), fused=True)


@pytest.mark.parametrize("heads,d,dtype", [(4, 64, "f32"), (16, 64, "f32"), (16, 64, "bf16"), (6, 50, "f32"), (6, 50, "bf16"), (8, 40, "bf16"), (3, 17, "f32"),
                                           (12, 64, "bf16"), (1, 1, "f32"), (1, 64, "bf16")])
@pytest.mark.parametrize("kind", [("bpt", 300, 4), ("memory", 5, 200)], ids=str)
def test_head_shapes(kind, heads, d, dtype):
    check(make(kind, heads, d, dtype), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 64, 65, 300, 1000])
def test_numbers_of_buckets(n, dtype):
    check(make(("bpt", 900, 4), 8, 64, dtype, n=n), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", [("bpt", 5000, 4), ("window", 4096, 64)], ids=str)
def test_graphs_that_fill_the_chip(kind, dtype):
    check(make(kind, 8, 64, dtype, n=32), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d", [(8, 64), (6, 50)])
@pytest.mark.parametrize("cap,distance", [(30.0, False), (15.0, True), (0.0, True)])
def test_with_score_options(heads, d, cap, distance, dtype):
    check(make(("bpt", 300, 4), heads, d, dtype, cap=cap, distance=distance), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d,kind,cap", [(8, 64, ("bpt", 300, 4), 0.0), (6, 50, ("random", 90, 1500), 0.0), (16, 64, ("window", 2000, 40), 0.0), (8, 64, ("bpt", 300, 4), 20.0)],
                         ids=str)
def test_dropout(heads, d, kind, cap, dtype):
    from bpt_amd import graphop
    c = make(kind, heads, d, dtype, cap=cap)
    hp = graphop.score_padded_shape(c["q"])[0]
    mask = graphop.attention_dropout_mask(None, None, c["src"], None, torch.empty(1, hp, 64), None, 0.2, 77)[:, :heads]
    check(c, fused=True, drop=mask.double(), dropout_p=0.2, seed=77)


@pytest.mark.parametrize("distance", [False, True])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_hidden_buckets_and_rows_with_nothing_left(dtype, fused, distance):
    """-infinity hides a bucket's edges: rows all of whose edges are hidden are 0 and have no gradient.  (Not a bucket that nothing is left of: its sum of ds is 0.)"""
    c = make(("random", 90, 400), 8, 64, dtype, n=4, distance=distance)
    c["bias_table"][1] = -math.inf
    c["buckets"][c["dst"] < 20] = 1
    args, got = check(c, fused=fused)
    assert not got["o"][:20].any() and not got["dq"][:20].any() and not got["dbias_table"][1].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_plans_built_on_the_host(dtype):
    from bpt_amd import plan
    old = plan.set_device_build(False)
    try:
        check(make(("bpt", 400, 4), 8, 64, dtype), fused=True)
    finally:
        plan.set_device_build(old)


def test_a_cache_too_small_for_the_plans():
    from bpt_amd.plan import plan_cache
    old = plan_cache._cap, plan_cache._max_bytes
    plan_cache.set_limits(1, 1)
    try:
        check(make(("bpt", 300, 4), 8, 64, "f32"), fused=True)
    finally:
        plan_cache.set_limits(*old)


@pytest.mark.parametrize("heads,d,dtype", [(2, 80, "f32"), (17, 8, "f32"), (8, 64, "f32"), (70, 4, "f32"), (3, 5, "f64")])
@pytest.mark.parametrize("kind", [("bpt", 60, 2), ("random", 90, 1500), ("memory", 5, 40)], ids=str)
def test_the_chain_of_operators(kind, heads, d, dtype):
    check(make(kind, heads, d, dtype), fused=False if d == 64 else None)


@pytest.mark.parametrize("switch", ["set_force_generic", "set_tiles", "set_row_groups"])
def test_kernels_switched_off(switch):
    from bpt_amd import graphop
    c = make(("bpt", 100, 4), 8, 64, "f32")
    old = getattr(graphop, switch)(switch == "set_force_generic")
    try:
        check(c)
    finally:
        getattr(graphop, switch)(False if switch == "set_force_generic" else old)


def test_units_that_leave_edges_out():
    """Edges that no unit covers take no part: they have no gradient either."""
    from bpt_amd import op
    c = make(("random", 90, 1500), 8, 64, "f32")
    args = list(graph_args(c["src"].numpy(), c["dst"].numpy(), 90, 90))
    # the in-side without its last unit, the out-side without the edges of that unit
    last = args[6][args[5][-2]:]
    args[4], args[5] = args[4][:-1].contiguous(), args[5][:-1].contiguous()
    keep = torch.ones(1500, dtype=torch.bool, device=DEV)
    keep[last] = False
    part = {n: t[keep.cpu()] if n in ("src", "dst", "buckets") else t for n, t in c.items()}
    want = reference(part)["o"]
    dev = on_device(c, False)
    close(call(c, dev, args), want, "o", torch.float32)


def test_the_separate_operator():
    from bpt_amd import op
    for dtype in (torch.float32, torch.float64, torch.bfloat16):
        for n, h, E in ((1, 1, 1), (7, 3, 1000), (200, 8, 5000), (40, 100, 3000), (600, 64, 777), (5, 8, 0)):
            gen = torch.Generator().manual_seed(n)
            table = torch.randn(n, h, generator=gen, dtype=torch.float64).to(dtype).to(DEV).requires_grad_(True)
            buckets, g = torch.randint(-1, n + 1, (E,), generator=gen).to(DEV), torch.randn(E, h, generator=gen, dtype=torch.float64).to(dtype).to(DEV)
            there = (buckets >= 0) & (buckets < n)
            y = op.bucket_bias(table, buckets)
            rows = table.detach()[torch.where(there, buckets, 0)]
            assert torch.equal(y, torch.where(there[:, None], rows, torch.zeros_like(rows)))
            (d,) = torch.autograd.grad(y, table, g)
            sums = torch.zeros(n + 1, h, dtype=torch.float64, device=DEV).index_add(0, torch.where(there, buckets, n), g.double())[:n]
            mags = torch.zeros(n + 1, h, dtype=torch.float64, device=DEV).index_add(0, torch.where(there, buckets, n), g.double().abs())[:n]
            half = torch.finfo(dtype).eps / 2
            assert ((d.double() - sums).abs() <= (E / 4096 + 600) * min(2.0 ** -24, half) * mags + half * sums.abs()).all()


def test_replays_of_a_captured_pass_match_the_eager_one():
    c = make(("bpt", 700, 4), 8, 64, "f32")
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c)
    leaves = [dev[n] for n in LEAVES if n in dev]

    def step():
        o = call(c, dev, args)
        return (o.detach(),) + torch.autograd.grad(o, leaves, dev["do"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, again)) and all(torch.equal(a, b) for a, b in zip(eager, step()))
    captured_graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured_graph):
        captured = step()
    for i in range(4):
        fresh = make(("bpt", 700, 4), 8, 64, "f32", seed=i + 1)
        with torch.no_grad():
            for n in ("q", "k", "v", "do", "bias_table", "buckets"):
                dev[n].copy_(fresh[n])
        captured_graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def test_no_edges_and_no_rows():
    from bpt_amd import op
    e = torch.empty(0, dtype=torch.int64, device=DEV)
    z = torch.zeros(1, dtype=torch.int64, device=DEV)
    q, k, v = (torch.randn(5, 8, 64, device=DEV, requires_grad=True) for _ in range(3))
    table = torch.ones(3, 8, device=DEV, requires_grad=True)
    o = op.bpt_attention(e, z, e, e, e, z, e, e, q, k, v, bias_table=table, buckets=e)
    grads = torch.autograd.grad(o, (q, k, v, table), torch.ones_like(o))
    assert o.shape == q.shape and not o.any() and not any(g.any() for g in grads)


def test_zero_bias_is_the_plain_layer_and_a_constant_moves_nothing():
    from bpt_amd import op
    c = make(("bpt", 300, 4), 8, 64, "f32")
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c, False)
    plain = op.bpt_attention(*args, dev["q"], dev["k"], dev["v"])
    for value in (0.0, 3.0):
        o = op.bpt_attention(*args, dev["q"], dev["k"], dev["v"], bias_table=torch.full((20, 8), value, device=DEV), buckets=dev["buckets"].clamp(0, 19))
        assert (o - plain).abs().max() < 1e-5


def test_a_second_derivative_is_refused():
    c = make(("bpt", 30, 2), 8, 64, "f32")
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c)
    with pytest.raises(RuntimeError, match="differentiable twice"):
        torch.autograd.grad(call(c, dev, args), dev["q"], dev["do"], create_graph=True)


def test_refusals():
    from bpt_amd import op
    c = make(("bpt", 30, 2), 8, 64, "f32")
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c, False)
    t, b = dev["bias_table"], dev["buckets"]
    go = lambda **kw: op.bpt_attention(*args, dev["q"], dev["k"], dev["v"], **kw)
    for match, exc, kw in [("go together", ValueError, dict(bias_table=t)), ("go together", ValueError, dict(buckets=b)),
                           ("bias_table must be", ValueError, dict(bias_table=t[:, :4].contiguous(), buckets=b)),
                           ("bias_table must be", ValueError, dict(bias_table=t[:0], buckets=b)), ("bias_table must be", ValueError, dict(bias_table=t[0], buckets=b)),
                           ("one element for every edge", ValueError, dict(bias_table=t, buckets=b[:-1])), ("int64", ValueError, dict(bias_table=t, buckets=b.int())),
                           ("one dtype", RuntimeError, dict(bias_table=t.bfloat16(), buckets=b)), ("one device", ValueError, dict(bias_table=t.cpu(), buckets=b)),
                           ("one device", ValueError, dict(bias_table=t, buckets=b.cpu())),
                           ("do not go together", ValueError, dict(bias_table=t, buckets=b, rel_table=torch.randn(3, 64, device=DEV), etype=b.clamp(0, 2)))]:
        with pytest.raises(exc, match=match):
            go(**kw)
    with pytest.raises(RuntimeError, match="no fused kernel"):
        op.bpt_attention(*args, *(torch.randn(c["q"].size(0), 2, 80, device=DEV) for _ in range(3)), fused=True, bias_table=t[:, :2].contiguous(), buckets=b)
    strided = go(bias_table=t.t().contiguous().t(), buckets=torch.stack([b, b], 1)[:, 0].contiguous())
    assert torch.equal(strided, go(bias_table=t, buckets=b))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [255, 256])
def test_as_many_buckets_as_a_byte_counts(n, dtype):
    check(make(("bpt", 900, 4), 8, 64, dtype, n=n), fused=True)


@pytest.mark.parametrize("scale", [-0.2, 1.5])
@pytest.mark.parametrize("heads,d,dtype", [(8, 64, "f32"), (6, 50, "bf16")])
def test_scales(heads, d, dtype, scale):
    """The bias is added behind the scale, whatever its sign and size."""
    from bpt_amd import op
    c = make(("bpt", 300, 4), heads, d, dtype)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c)
    o = call(c, dev, args, scale=scale)
    e = (dev["q"].double()[c["dst"].to(DEV)] * dev["k"].double()[c["src"].to(DEV)]).sum(-1) * scale
    b = c["buckets"].to(DEV)
    there = (b >= 0) & (b < 20)
    e = e + torch.where(there[:, None], dev["bias_table"].double()[torch.where(there, b, 0)], 0.0)
    dst, src = c["dst"].to(DEV), c["src"].to(DEV)
    w = torch.exp(e - e.max())
    total = torch.zeros(c["q"].size(0), heads, dtype=torch.float64, device=DEV).index_add(0, dst, w)
    want = torch.zeros(o.shape, dtype=torch.float64, device=DEV).index_add(0, dst, (w / total[dst])[:, :, None] * dev["v"].double()[src])
    half = torch.finfo(c["q"].dtype).eps / 2
    # 300 terms of a row at most: scores up to 40 with 72 2^-24 of the products' absolute values twice, p and o rounded once each
    assert ((o.double() - want).abs() <= (2 * half + 2.0 ** -13) * (1 + dev["v"].abs().max().double())).all()
    got = torch.autograd.grad(o, [dev[n] for n in ("q", "k", "v", "bias_table")], dev["do"])
    ref = torch.autograd.grad(want, [dev[n] for n in ("q", "k", "v", "bias_table")], dev["do"].double())
    for x, y in zip(got, ref):
        assert (x.double() - y.double()).norm() <= (8 * half + 2.0 ** -12) * y.double().norm()


def test_some_of_the_gradients():
    c = make(("bpt", 300, 4), 8, 64, "f32", distance=True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    everything = run(c, args)
    for names in (["bias_table"], ["slopes"], ["q"], ["v", "bias_table"], ["k", "slopes"]):
        dev = {n: t.to(DEV).requires_grad_(n in names) for n, t in c.items() if torch.is_tensor(t)}
        o = call(c, dev, args)
        for n, g in zip(names, torch.autograd.grad(o, [dev[n] for n in names], dev["do"])):
            assert torch.equal(g, everything["d" + n]), n


def test_views_and_saved_tensors_that_went_elsewhere():
    c = make(("bpt", 300, 4), 8, 64, "f32", distance=True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    want = run(c, args)
    dev = on_device(c)
    leaves = [dev[n] for n in LEAVES if n in dev]
    names = ["d" + n for n in LEAVES if n in dev]
    wide = torch.stack((dev["buckets"], dev["buckets"]), 1)
    views = dict(dev, bias_table=dev["bias_table"].t().contiguous().t(), buckets=wide[:, 1])
    assert not views["bias_table"].is_contiguous() and not views["buckets"].is_contiguous()
    o = call(c, views, args)
    grads = torch.autograd.grad(o, leaves, dev["do"], retain_graph=True)
    assert torch.equal(o, want["o"]) and all(torch.equal(g, want[n]) for n, g in zip(names, grads))
    assert all(torch.equal(g, want[n]) for n, g in zip(names, torch.autograd.grad(o, leaves, dev["do"])))
    with torch.autograd.graph.save_on_cpu():
        o = call(c, dev, args)
    grads = torch.autograd.grad(o, leaves, dev["do"].transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(g, want[n]) for n, g in zip(names, grads))
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x.double() if x.is_floating_point() else x):
        o = call(c, dev, args)
    with pytest.raises(RuntimeError, match="saved tensors"):
        torch.autograd.grad(o, leaves, dev["do"])


def test_two_calls_of_one_graph_before_their_backwards():
    c, other = make(("bpt", 300, 4), 8, 64, "bf16"), make(("bpt", 300, 4), 8, 64, "bf16", seed=5)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    want = run(c, args), run(other, args)
    devs = on_device(c), on_device(other)
    outs = [call(x, d, args) for x, d in zip((c, other), devs)]
    for o, d, w in zip(outs, devs, want):
        names = [n for n in LEAVES if n in d]
        assert torch.equal(o, w["o"]) and all(torch.equal(g, w["d" + n]) for n, g in zip(names, torch.autograd.grad(o, [d[n] for n in names], d["do"])))


@pytest.mark.parametrize("how", ["fused", "long", "chain"])
@pytest.mark.parametrize("dtype,mask", [("f32", -2.0 ** 19), ("f32", -1e9), ("f32", torch.finfo(torch.float32).min), ("bf16", -1e6), ("bf16", torch.finfo(torch.bfloat16).min)])
def test_masks_of_large_numbers_hide(dtype, mask, how):
    """As -infinity: the same bits.  (long: a table of more buckets than the fastest path takes.)"""
    c = make(("random", 90, 400), 8, 64, dtype, n=300 if how == "long" else 4)
    c["buckets"][c["dst"] < 20] = 1
    c["bias_table"][1] = -math.inf
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    want = run(c, args, fused=how != "chain")
    c["bias_table"][1] = mask
    got = run(c, args, fused=how != "chain")
    assert not got["o"][:20].any() and all(torch.equal(got[n], want[n]) and got[n].isfinite().all() for n in got)


@pytest.mark.parametrize("n", [4, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_cap_bounds_masks(dtype, n):
    c = make(("random", 90, 400), 8, 64, dtype, n=n, cap=15.0)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    c["bias_table"][1] = -3000.0                                  # (200 caps: the tangent is -1)
    want = run(c, args, fused=True)
    for mask in (-1e9, -math.inf, torch.finfo(c["q"].dtype).min):
        c["bias_table"][1] = mask
        got = run(c, args, fused=True)
        assert all(torch.equal(got[m], want[m]) for m in got), mask
