"""op.bpt_attention with capped scores and distance (score_cap, slopes, pos) against the formula in 64 bits.

Tolerances, from the arithmetic, per element.  E = 2^-24; F = half a step of the result's type beyond float32 (bfloat16 2^-8, else 0).
  score  u = scale q.k(+ term): 64 products and their sum, 72 E of the sum of absolute values (a second such sum for the term, which is stored
         once); tanh 3 E relative, the cap's factor, the change to base 2, the distance's product and the difference to lse: 12 E of the absolute
         values of what is added, with lse
  p      relative: exp2 of that (the error in natural units) once for the pair and once for the row's sum, and (edges of the row + 16) E for the sum
  o      the relative error of p twice over sum p |v| (numerator and denominator), (edges + 16) E of it, F for p rounded on its way into the product
  dp, delta   72 E of the sums of absolute values; delta uses o as stored (F of sum |dO| |o| more)
  ds     p's relative error of p (|dp| + |delta|), those two errors times p; du: (1 - t^2) is off by 8 E, F for du rounded on its way
  dq, dk, dv  sums of such terms over edges: their bounds' sums and (edges + 16) E of the sum of absolute values
  dslopes     the same over all edges; a lane adds at most edges / 16 + 64 of them in turn
and half a step of the result's type."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f64": torch.float64}


def graph(kind):
    """(src, dst, n_q, n_k) of edge lists: BPT graphs, windows, random multigraphs with empty rows and duplicate edges, attention to a memory."""
    from bpt_amd import graphbuilder as gb
    name, *num = kind
    rng = np.random.default_rng(sum(num))
    if name == "bpt":
        g = gb.BinaryPartition(num[0], True, num[1], 10)
        src, dst, _ = g.get_edges()
        return src, dst, g.number_of_nodes, g.number_of_nodes
    if name == "window":
        g = gb.FullyConnected(num[0], True, num[1])
        src, dst, _ = g.get_edges()
        return src, dst, g.number_of_nodes, g.number_of_nodes
    if name == "random":                                          # num: nodes, edges; the last third of the nodes has no in-edges
        return rng.integers(0, num[0], num[1]), rng.integers(0, max(1, num[0] * 2 // 3), num[1]), num[0], num[0]
    n_q, n_k = num                                                # "memory"
    return np.tile(np.arange(n_k), n_q), np.repeat(np.arange(n_q), n_k), n_q, n_k


def graph_args(src, dst, n_q, n_k):
    from bpt_amd import graphbuilder as gb
    csr = gb.get_csrs(src, dst, n_q) if n_q == n_k else gb.get_csrs_bipartite(src, dst, n_k, n_q)
    out_csr, in_csr, row, ir, col, ic = csr
    return tuple(t.to(DEV) for t in (row, ir, out_csr[2], out_csr[1], col, ic, in_csr[2], in_csr[1]))


def make(kind, heads, d, dtype, cap, distance, rel=False, seed=0, q_scale=1.0):
    src, dst, n_q, n_k = graph(kind)
    gen = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    rand = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)
    c = dict(src=torch.from_numpy(np.asarray(src, dtype=np.int64)), dst=torch.from_numpy(np.asarray(dst, dtype=np.int64)), cap=cap,
             q=(rand(n_q, heads, d) * q_scale).to(t), k=rand(n_k, heads, d).to(t), v=rand(n_k, heads, d).to(t), do=(rand(n_q, heads, d) / 8).to(t))
    if distance:
        c["slopes"] = (2.0 ** (-8.0 * torch.arange(1, heads + 1) / heads) * (1 + 0.1 * rand(heads).abs())).float()
        c["pos_q"] = torch.sort(rand(n_q) * n_q).values.float()
        c["pos_k"] = c["pos_q"] if n_q == n_k else torch.sort(rand(n_k) * n_k).values.float()
    if rel:
        c["table"] = (rand(30, d) * 0.3).to(t)
        c["etype"] = torch.from_numpy(np.random.default_rng(5).integers(0, 30, len(src)))
    return c


def reference(c, drop=None):
    """{name: (value, bound)} in 64 bits."""
    src, dst = c["src"], c["dst"]
    D = {n: t.double() for n, t in c.items() if torch.is_tensor(t) and t.is_floating_point()}
    q, k, v, do = (D[n] for n in ("q", "k", "v", "do"))
    n_q, h, d = q.shape
    n_e, scale, cap, E = src.numel(), 1 / math.sqrt(d), c["cap"], 2.0 ** -24
    F = 2.0 ** -8 if c["q"].dtype == torch.bfloat16 else 0.0
    seg = lambda x, to, n: torch.zeros((n,) + x.shape[1:], dtype=torch.float64).index_add(0, to, x)
    qe, ke, ve, doe = q[dst], k[src], v[src], do[dst]
    x, ax = (qe * ke).sum(-1), (qe * ke).abs().sum(-1)
    if "table" in c:
        te = D["table"][c["etype"]][:, None]
        x, ax = x + (qe * te).sum(-1), ax + 2 * (qe * te).abs().sum(-1)
    u, du_err = x * scale, 72 * E * ax * scale
    t = torch.tanh(u / cap) if cap else None
    s = cap * t if cap else u
    slope = 1 - t * t if cap else torch.ones_like(u)
    mag = s.abs()
    far = None
    if "slopes" in c:
        far = (D["pos_q"][dst] - D["pos_k"][src]).abs()[:, None]
        s = s - D["slopes"] * far
        mag = mag + D["slopes"] * far
    idx = dst[:, None].expand(-1, h)
    top = torch.full((n_q, h), -1e300, dtype=torch.float64).scatter_reduce(0, idx, s, "amax")
    w = torch.exp(s - top[dst])
    total = seg(w, dst, n_q)
    p = w / total[dst]
    lse = torch.log(total.clamp(min=1e-300)) + top
    err_s = du_err + 12 * E * (mag + lse[dst].abs())
    deg = torch.zeros(n_q, dtype=torch.float64).index_add(0, dst, torch.ones(n_e, dtype=torch.float64))
    row_err = torch.zeros((n_q, h), dtype=torch.float64).scatter_reduce(0, idx, err_s, "amax")
    rho = err_s + row_err[dst] + (deg[dst] + 16)[:, None] * E      # relative, of p
    m = drop if drop is not None else torch.ones_like(p)
    o = seg((p * m)[..., None] * ve, dst, n_q)
    o_b = seg((p * m * (2 * rho + F))[..., None] * ve.abs(), dst, n_q) + (deg + 16)[:, None, None] * E * seg((p * m)[..., None] * ve.abs(), dst, n_q)
    dp, adp = (doe * ve).sum(-1), (doe * ve).abs().sum(-1)
    delta, adelta = (do * o).sum(-1), (do * o).abs().sum(-1)
    delta_b = 72 * E * adelta + F * adelta + (do.abs() * o_b).sum(-1)
    ds = p * (dp * m - delta[dst])
    ds_b = p * (rho * (dp.abs() * m + delta.abs()[dst]) + 72 * E * adp * m + delta_b[dst])
    du = ds * slope * scale
    du_b = (ds_b * slope + ds.abs() * 8 * E + F * (ds * slope).abs() + 4 * E * (ds * slope).abs()) * scale
    out = {"o": (o, o_b)}
    deg_k = torch.zeros(k.size(0), dtype=torch.float64).index_add(0, src, torch.ones(n_e, dtype=torch.float64))
    ks = ke + (te if "table" in c else 0.0)
    pm, pm_b = p * m, p * m * (rho + F)
    for name, to, n, g, a, a_b, y in (("dq", dst, n_q, deg, du, du_b, ks), ("dk", src, k.size(0), deg_k, du, du_b, qe), ("dv", src, k.size(0), deg_k, pm, pm_b, doe)):
        out[name] = (seg(a[..., None] * y, to, n), seg(a_b[..., None] * y.abs(), to, n) + (g + 16)[:, None, None] * E * seg(a.abs()[..., None] * y.abs(), to, n))
    if far is not None:
        out["dslopes"] = (-(ds * far).sum(0), (ds_b * far).sum(0) + (n_e / 16 + 64) * E * (ds * far).abs().sum(0))
    if "table" in c:
        per = (du[..., None] * qe).sum(1), (du_b[..., None] * qe.abs()).sum(1) + (n_e * h / 30 + 64) * E * (du.abs()[..., None] * qe.abs()).sum(1)
        out["dtable"] = tuple(seg(y, c["etype"], 30) for y in per)
        # dq is formed in two steps, sum ds k stored in the result's type, then read and sum ds table added: ds is rounded on its way into the first alone, and the
        # sum is once more where it is stored, F of sum |ds| |k| each (also where k and table cancel in sum ds (k + table), which the terms above go by), of ds as computed
        out["dq"] = (out["dq"][0], out["dq"][1] + F * out["dq"][0].abs() + 2 * F * seg((du.abs() + du_b)[..., None] * ke.abs(), dst, n_q))
    return out


def call(c, dev, args, fused=None, **kw):
    from bpt_amd import op
    opts = {}
    if c["cap"]:
        opts["score_cap"] = c["cap"]
    if "slopes" in c:
        opts.update(slopes=dev["slopes"], pos=dev["pos_q"] if c["pos_q"] is c["pos_k"] else (dev["pos_q"], dev["pos_k"]))
    if "table" in c:
        opts.update(rel_table=dev["table"], etype=dev["etype"])
    return op.bpt_attention(*args, dev["q"], dev["k"], dev["v"], fused=fused, **opts, **kw)


def on_device(c, grad=True):
    return {n: t.to(DEV).requires_grad_(grad and n in ("q", "k", "v", "slopes", "table")) for n, t in c.items() if torch.is_tensor(t)}


def close(got, want, name, dtype):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    excess = (got - value).abs() - bound - torch.finfo(dtype).eps / 2 * value.abs() - 1e-30
    assert not torch.isnan(got).any(), name
    assert excess.numel() == 0 or excess.max().item() <= 0, f"{name}: beyond its bound by {excess.max().item():.3e} (bound there {bound.flatten()[excess.argmax()].item():.3e})"


def run(c, args, fused=None, **kw):
    dev = on_device(c)
    o = call(c, dev, args, fused, **kw)
    names = ["q", "k", "v"] + [n for n in ("slopes", "table") if n in c]
    grads = torch.autograd.grad(o, [dev[n] for n in names], dev["do"])
    return dict({"o": o.detach()}, **{"d" + n: g for n, g in zip(names, grads)})


def check(c, fused=None, drop=None, **kw):
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    ref = reference(c, drop)
    for _ in range(2):                                            # (the second call is the one that finds what the first left)
        got = run(c, args, fused, **kw)
        for n, want in ref.items():
            close(got[n], want, n, torch.float32 if n == "dslopes" else c["q"].dtype)
    with torch.no_grad():
        o = call(c, on_device(c, False), args, fused, **kw)
        close(o, ref["o"], "o without gradients", c["q"].dtype)
    return args, got


OPTIONS = [(30.0, False), (0.0, True), (30.0, True), (1.0, True)]
GRAPHS = [("bpt", 1, 1), ("bpt", 5, 2), ("bpt", 33, 4), ("bpt", 700, 4), ("window", 300, 20), ("random", 90, 1500), ("random", 3, 5), ("random", 1000, 300),
          ("memory", 1, 700), ("memory", 17, 3), ("memory", 1, 1), ("memory", 40, 300)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap,distance", OPTIONS)
@pytest.mark.parametrize("kind", GRAPHS, ids=str)
def test_matches_the_formula(kind, cap, distance, dtype):
    check(make(kind, 8, 64, dtype, cap, distance), fused=True)


@pytest.mark.parametrize("heads,d,dtype", [(4, 64, "f32"), (16, 64, "f32"), (16, 64, "bf16"), (6, 50, "f32"), (6, 50, "bf16"), (8, 40, "bf16"), (3, 17, "f32"),
                                           (12, 64, "bf16"), (8, 32, "f32"), (1, 1, "f32"), (1, 64, "bf16"), (16, 63, "bf16")])
@pytest.mark.parametrize("kind", [("bpt", 300, 4), ("memory", 5, 200)], ids=str)
def test_head_shapes(kind, heads, d, dtype):
    check(make(kind, heads, d, dtype, 20.0, True), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_graph_that_fills_the_chip(dtype):
    check(make(("bpt", 5000, 4), 8, 64, dtype, 30.0, True), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d", [(8, 64), (6, 50)])
def test_tiles_in_two_parts_and_long_rows(heads, d, dtype):
    """About 2056 wavefronts (1542 of six heads) of five blocks: two wavefronts a tile; the last row has 4096 edges, in many segments."""
    check(make(("window", 4096, 64), heads, d, dtype, 30.0, True), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_plans_built_on_the_host(dtype):
    from bpt_amd import plan
    old = plan.set_device_build(False)
    try:
        check(make(("bpt", 400, 4), 8, 64, dtype, 30.0, True), fused=True)
    finally:
        plan.set_device_build(old)


def test_a_cache_too_small_for_the_plans():
    """Nothing is left with the native host path: the Python function runs, again and again."""
    from bpt_amd.plan import plan_cache
    old = plan_cache._cap, plan_cache._max_bytes
    plan_cache.set_limits(1, 1)
    try:
        check(make(("bpt", 300, 4), 8, 64, "f32", 30.0, True), fused=True)
        check(make(("bpt", 300, 4), 6, 50, "f32", 30.0, True), fused=True)
    finally:
        plan_cache.set_limits(*old)


def test_generic_kernels_forced():
    from bpt_amd import graphop
    c = make(("bpt", 100, 4), 8, 64, "f32", 30.0, True)
    args, _ = check(c)
    graphop.set_force_generic(True)
    try:
        check(c)
        with pytest.raises(RuntimeError, match="no fused kernel"):
            run(c, args, fused=True)
    finally:
        graphop.set_force_generic(False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [0.5, 4.0])
def test_saturated_scores(cap, dtype):
    """Scores of tens over a cap of few: tanh is +-1 and its derivative 0 to the last digit."""
    check(make(("bpt", 200, 4), 8, 64, dtype, cap, False, q_scale=20.0), fused=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d,kind,rel", [(8, 64, ("bpt", 300, 4), False), (6, 50, ("bpt", 300, 4), False), (6, 50, ("memory", 40, 300), False),
                                              (12, 64, ("window", 2000, 40), False), (8, 64, ("bpt", 300, 4), True), (6, 50, ("random", 90, 1500), True)], ids=str)
def test_dropout(heads, d, kind, rel, dtype):
    from bpt_amd import graphop
    c = make(kind, heads, d, dtype, 30.0, True, rel=rel)
    hp = graphop.score_padded_shape(c["q"])[0]
    mask = graphop.attention_dropout_mask(None, None, c["src"], None, torch.empty(1, hp, 64), None, 0.2, 77)[:, :heads]
    check(c, fused=True, drop=mask.double(), dropout_p=0.2, seed=77)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap,scale", [(1e-10, 1e-10), (1e10, 0.125), (1e10, 1e6), (0.0125, 125.0), (1e-10, 1e-6)])
def test_the_largest_and_smallest_caps(cap, scale, dtype):
    """Every value is an ordinary number there.  (q is scaled so that the scores are a few units or caps, whichever is less.)"""
    c = make(("bpt", 60, 2), 8, 64, dtype, 0.0, True, q_scale=min(0.125, cap) / scale)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c)
    from bpt_amd import op
    o = op.bpt_attention(*args, dev["q"], dev["k"], dev["v"], scale=scale, score_cap=cap, slopes=dev["slopes"], pos=dev["pos_q"], fused=True)
    grads = torch.autograd.grad(o, [dev["q"], dev["k"], dev["v"], dev["slopes"]], dev["do"])
    chain = op.bpt_attention(*args, *(dev[n].double() for n in ("q", "k", "v")), scale=scale, score_cap=cap, slopes=dev["slopes"], pos=dev["pos_q"])
    want = torch.autograd.grad(chain, [dev["q"], dev["k"], dev["v"], dev["slopes"]], dev["do"].double())
    # F: o, and ds and p on their way into a product and the result, half a step each of the norm; float32's roundings are far below 2e-5 of the norm here
    F = 4 * 2.0 ** -8 if dtype == "bf16" else 2e-5
    for name, got, ref in zip(("o", "dq", "dk", "dv", "dslopes"), (o, *grads), (chain, *want)):
        assert got.isfinite().all() and (got.double() - ref.double()).norm() <= F * ref.double().norm(), (name, (got.double() - ref.double()).norm() / ref.double().norm())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d", [(8, 64), (16, 64), (6, 50)])
@pytest.mark.parametrize("cap,distance", [(30.0, False), (15.0, True)])
def test_with_relative_positions(heads, d, cap, distance, dtype):
    check(make(("bpt", 300, 4), heads, d, dtype, cap, distance, rel=True), fused=True)


@pytest.mark.parametrize("heads,d,dtype", [(2, 80, "f32"), (17, 8, "f32"), (8, 64, "f32")])
@pytest.mark.parametrize("kind", [("bpt", 60, 2), ("random", 90, 1500), ("memory", 5, 40)], ids=str)
def test_the_chain_of_operators(kind, heads, d, dtype):
    """Shapes without a fused kernel, and fused=False.  E holds for the chain's roundings too: each tensor between its operators is one more."""
    check(make(kind, heads, d, dtype, 20.0, True), fused=False if d == 64 else None)


def test_the_chain_in_64_bits_against_differences():
    from bpt_amd import op
    c = make(("random", 12, 60), 2, 5, "f64", 2.0, True, rel=True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), 12, 12)
    dev = on_device(c)
    slopes = dev["slopes"].detach().double().requires_grad_(True)
    f = lambda q, k, v, s: op.bpt_attention(*args, q, k, v, score_cap=2.0, slopes=s.float(), pos=dev["pos_q"])
    assert torch.autograd.gradcheck(lambda q, k, v: f(q, k, v, slopes.detach()), (dev["q"], dev["k"], dev["v"]))


def test_gradients_against_differences():
    """Float32: the central difference of sum(dO o) along a random direction, step 2^-6: truncation of the order of the step squared, rounding of sums of n
    terms divided by the step; both are below 2 % of the derivative's scale here, which is what is asked."""
    c = make(("bpt", 40, 2), 8, 64, "f32", 5.0, True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    got, step = run(c, args), 2.0 ** -6
    for n in ("q", "k", "v", "slopes"):
        way = torch.randn(c[n].shape, generator=torch.Generator().manual_seed(9))
        way = way / way.norm()
        value = []
        for sign in (1, -1):
            moved = dict(c, **{n: c[n] + sign * step * way})
            with torch.no_grad():
                value.append((call(moved, on_device(moved, False), args).double() * c["do"].to(DEV).double()).sum())
        want = ((value[0] - value[1]) / (2 * step)).item()
        have = (got["d" + n].cpu().double() * way.double()).sum().item()
        assert abs(have - want) <= 0.02 * max(abs(want), got["d" + n].norm().item() / way.numel() ** 0.5), (n, have, want)


def close_where_finite(got, want, name, dtype):
    """As close(), of results that are infinite or NaN where the formula's are, and only there."""
    value, bound = want
    got = got.detach().cpu().double()
    fine = value.isfinite()
    assert torch.equal(got.isfinite(), fine), f"{name}: {int((~got.isfinite() & fine).sum())} of {int(fine.sum())} finite results are not, {int((got.isfinite() & ~fine).sum())} are that must not be"
    if fine.any():
        close(got[fine], (value[fine], bound[fine]), name, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d,rel", [(8, 64, False), (6, 50, False), (8, 64, True)])
@pytest.mark.parametrize("kind", [("bpt", 300, 4), ("random", 1000, 300), ("memory", 40, 300), ("bpt", 5000, 4)], ids=str)
@pytest.mark.parametrize("where", ["v", "k", "q", "do", "pos"])
def test_what_stands_in_rows_that_are_not_neighbours(where, kind, heads, d, rel, dtype):
    """One row (the last of the second third; of positions, one without edges) is infinite in its first column and NaN in its second."""
    c = make(kind, heads, d, dtype, 30.0, True, rel=rel)
    c = {n: t.clone() if torch.is_tensor(t) and n not in ("pos_q", "pos_k") else t for n, t in c.items()}
    if where == "pos":
        lone = np.setdiff1d(np.arange(c["q"].size(0)), np.concatenate([c["dst"].numpy(), c["src"].numpy()] if c["q"].size(0) == c["k"].size(0) else [c["dst"].numpy()]))
        if not len(lone):
            pytest.skip("every row has edges")
        same = c["pos_q"] is c["pos_k"]
        c["pos_q"] = c["pos_q"].clone()
        c["pos_q"][torch.from_numpy(lone)] = torch.tensor([float("inf"), float("nan")]).repeat(len(lone))[:len(lone)]
        if same:
            c["pos_k"] = c["pos_q"]
    else:
        row = c[where].size(0) * 2 // 3 - 1
        c[where][row, :, 0], c[where][row, :, 1] = float("inf"), float("nan")
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    ref = reference(c)
    got = run(c, args, True)
    for n, want in ref.items():
        close_where_finite(got[n], want, n, torch.float32 if n == "dslopes" else c["q"].dtype)


def test_without_options_is_the_plain_layer():
    """A cap far beyond the scores and slopes of zero: the plain layer's numbers to rounding."""
    from bpt_amd import op
    c = make(("bpt", 600, 4), 8, 64, "f32", 3.0e4, True)
    c["slopes"] = torch.zeros(8)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c, False)
    plain = op.bpt_attention(*args, dev["q"], dev["k"], dev["v"])
    assert (call(c, dev, args) - plain).abs().max() < 1e-5


def test_the_same_bits_every_time_and_on_another_stream():
    c = make(("bpt", 900, 4), 8, 64, "f32", 30.0, True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    first = run(c, args)
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            again = run(c, args)
        torch.cuda.synchronize()
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_rows_off_16_bytes():
    c = make(("bpt", 100, 2), 8, 64, "f32", 30.0, True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    want = run(c, args)
    dev = on_device(c)
    for n in ("q", "k", "v", "do", "pos_q", "slopes"):
        buf = torch.empty(dev[n].numel() + 1, device=DEV)
        dev[n] = buf[1:].view(dev[n].shape).copy_(dev[n].detach()).detach().requires_grad_(dev[n].requires_grad)
    o = call(c, dev, args)
    grads = torch.autograd.grad(o, [dev[n] for n in ("q", "k", "v", "slopes")], dev["do"])
    assert torch.equal(o.detach(), want["o"]) and all(torch.equal(g, want[n]) for n, g in zip(("dq", "dk", "dv", "dslopes"), grads))


def test_no_edges_and_no_rows():
    from bpt_amd import op
    e = torch.empty(0, dtype=torch.int64, device=DEV)
    z = torch.zeros(1, dtype=torch.int64, device=DEV)
    args = (e, z, e, e, e, z, e, e)
    q, k, v = (torch.randn(5, 8, 64, device=DEV, requires_grad=True) for _ in range(3))
    slopes = torch.ones(8, device=DEV, requires_grad=True)
    o = op.bpt_attention(*args, q, k, v, score_cap=3.0, slopes=slopes, pos=torch.arange(5.0, device=DEV))
    grads = torch.autograd.grad(o, (q, k, v, slopes), torch.ones_like(o))
    assert o.shape == q.shape and not o.any() and not any(g.any() for g in grads)


def test_far_positions_and_negative_slopes():
    """Distances of 10^6 leave only the nearest; a negative slope prefers the farthest.  -slope |distance| is exact to E of itself, which at 10^6 is
    what a score is off by: 0.06 times the slope, so the neighbours' distances differ by far more."""
    from bpt_amd import op
    src, dst, n, _ = graph(("window", 64, 5))
    args = graph_args(src, dst, n, n)
    q, k, v = (torch.randn(n, 8, 64, device=DEV) for _ in range(3))
    pos = torch.arange(n, device=DEV).float() * 1e6
    for sign in (1.0, -1.0):
        o = op.bpt_attention(*args, q, k, v, score_cap=10.0, slopes=torch.full((8,), sign, device=DEV), pos=pos)
        for i in range(n):
            near = src[dst == i]
            far = np.abs(near - i)
            pick = near[far.argmin() if sign > 0 else far.argmax()] if len(near) else None
            want = torch.zeros(8, 64) if pick is None else v[int(pick)].cpu()
            assert torch.equal(o[i].cpu(), want), i


def test_replays_of_a_captured_pass_match_the_eager_one():
    c = make(("bpt", 700, 4), 8, 64, "f32", 30.0, True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c)
    leaves = [dev[n] for n in ("q", "k", "v", "slopes")]

    def step():
        o = call(c, dev, args)
        return (o.detach(),) + torch.autograd.grad(o, leaves, dev["do"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    captured_graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured_graph):
        captured = step()
    for i in range(4):
        fresh = make(("bpt", 700, 4), 8, 64, "f32", 30.0, True, seed=i + 1)
        with torch.no_grad():
            for n in ("q", "k", "v", "do", "slopes"):
                dev[n].copy_(fresh[n])
        captured_graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


@pytest.mark.parametrize("heads,d,kind,rel", [(h, d, kind, False) for h, d in ((8, 64), (16, 64), (6, 50)) for kind in (("bpt", 700, 4), ("memory", 71, 774), ("window", 1500, 40))]
                         + [(h, d, kind, True) for h, d in ((8, 64), (6, 50)) for kind in (("random", 900, 15000), ("memory", 71, 774))], ids=str)
def test_slopes_of_bfloat16_rows_are_summed_in_32_bits(heads, d, kind, rel):
    """Nothing that the slopes' gradient is summed from is rounded to bfloat16 (delta comes from the pairs): float32's bound, of the same values.  With a score term this
    holds where no row is split or half of them are."""
    c = make(kind, heads, d, "bf16", 15.0, True, rel=rel)
    wide = {n: t.float() if torch.is_tensor(t) and t.dtype == torch.bfloat16 else t for n, t in c.items()}
    got = run(c, graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0)), True)
    close(got["dslopes"], reference(wide)["dslopes"], "dslopes", torch.float32)


@pytest.mark.parametrize("rel", [False, True])
def test_a_second_derivative_is_refused(rel):
    c = make(("bpt", 30, 2), 8, 64, "f32", 30.0, True, rel=rel)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c)
    with pytest.raises(RuntimeError, match="differentiable twice"):
        torch.autograd.grad(call(c, dev, args), dev["q"], dev["do"], create_graph=True)


def test_refusals():
    from bpt_amd import op
    c = make(("bpt", 30, 2), 8, 64, "f32", 30.0, True)
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    dev = on_device(c, False)
    go = lambda **kw: op.bpt_attention(*args, dev["q"], dev["k"], dev["v"], **kw)
    for opts in (dict(score_cap=3.0), dict(slopes=dev["slopes"], pos=dev["pos_q"])):      # (what follows is refused of a graph that is known, too)
        go(**opts), go(**opts)
    for cap in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="score_cap"):
            go(score_cap=cap)
    with pytest.raises(ValueError, match="pair"):
        go(slopes=dev["slopes"], pos=(dev["pos_q"],))
    with pytest.raises(ValueError, match="at least"):
        go(score_cap=1e-6)
    with pytest.raises(ValueError, match="go together"):
        go(slopes=dev["slopes"])
    with pytest.raises(ValueError, match="go together"):
        go(pos=dev["pos_q"])
    with pytest.raises(ValueError, match="slopes must have shape"):
        go(slopes=dev["slopes"][:4].contiguous(), pos=dev["pos_q"])
    with pytest.raises(ValueError, match="pos .of the key rows. must have shape"):
        go(slopes=dev["slopes"], pos=(dev["pos_q"], dev["pos_k"][:3].contiguous()))
    with pytest.raises(RuntimeError, match="float32"):
        go(slopes=dev["slopes"], pos=dev["pos_q"].double())
    with pytest.raises(RuntimeError, match="CUDA"):
        go(slopes=dev["slopes"].cpu(), pos=dev["pos_q"])
    with pytest.raises(ValueError, match="no gradient"):
        go(slopes=dev["slopes"], pos=dev["pos_q"].clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="no fused kernel"):
        op.bpt_attention(*args, *(torch.randn(c["q"].size(0), 2, 80, device=DEV) for _ in range(3)), fused=True, score_cap=3.0)
