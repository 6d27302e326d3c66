"""What the operators around and inside a block's attention are measured on: passes through the public entry points, and the same
passes in elementary torch operations.

A case is a dict of plain values; `op` names the operator:

  "attention"  op.bpt_attention with the scores of an edge u = scale q[dst].k[src] capped to `cap` tanh(u / cap) (0: not capped) and, with
               `distance`, lowered by slopes[head] |pos[dst] - pos[src]|.  `graph`: "bpt" a causal binary-partition graph of `length` tokens,
               `k` neighbours per level; "window" every token attends to the `k` tokens before it and itself; "memory" `k` query rows that
               attend to all of `length` key rows.  `heads`, `d`; dtype "f32" or "bf16"; `backward`: with the gradients of q, k, v and slopes
  "norm"       op.add_layer_norm of `rows` rows of `cols` columns; `residual`: of a sum of two tensors; `backward`: with all gradients
  "relu8"      graphop.relu8_forward and relu8_backward of `rows` x `cols` activations: relu, its result kept in 8 bits, and the gradient

Node features are N(0, 1), as projections of layer-normalised states are, incoming gradients N(0, 1) / 8; slopes fall by heads from 2^(-8/h)
to 2^-8, as trained ones start.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 64              # activations that share a step


def _attention(graph, length, k, heads=8, d=64, dtype="f32", cap=0.0, distance=False, backward=True, name=None):
    c = dict(op="attention", graph=graph, length=length, k=k, heads=heads, d=d, dtype=dtype, cap=cap, distance=distance, backward=backward)
    return c if name is None else dict(c, name=name)


def _norm(rows, cols, dtype="f32", residual=True, backward=True, name=None):
    c = dict(op="norm", rows=rows, cols=cols, dtype=dtype, residual=residual, backward=backward)
    return c if name is None else dict(c, name=name)


def _relu8(rows, cols, dtype="f32", name=None):
    c = dict(op="relu8", rows=rows, cols=cols, dtype=dtype)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a decoder that takes one new token: its row attends to a memory of 2048 nodes
        _attention("memory", 2048, 1, cap=30.0, distance=True, backward=False, name="attend-row2048-f32"),
        # one paragraph-sized sequence in training
        _attention("bpt", 512, 4, cap=30.0, distance=True, name="attend-L512-f32"),
        # a character-level language model's layer, 8192 tokens of context
        _attention("bpt", 8192, 4, cap=30.0, distance=True, name="attend-L8192-f32"),
        # local attention, scores capped only: the densest neighbourhoods, narrow heads of the classification configurations
        _attention("window", 4096, 128, heads=6, d=50, cap=50.0, name="attend-L4096-w128-6x50-f32"),
        # the largest: long context, wide neighbourhood, 16 heads
        _attention("bpt", 32768, 8, heads=16, dtype="bf16", cap=30.0, distance=True, name="attend-L32768-k8-bf16"),
        # one token of a trained model
        _norm(1, 512, backward=False, name="norm-1x512-f32"),
        # a classification batch of 6 heads x 50 columns
        _norm(33598, 300, name="norm-33598x300-f32"),
        # the nodes of one sequence of 8192 tokens
        _norm(16383, 512, name="norm-16383x512-f32"),
        # those of 32768 tokens
        _norm(65535, 1024, dtype="bf16", name="norm-65535x1024-bf16"),
        # feed-forwards of four times the model's width, of 512, 8192 and 32768 tokens
        _relu8(1023, 2048, name="relu8-1023x2048-f32"),
        _relu8(16383, 2048, name="relu8-16383x2048-f32"),
        _relu8(65535, 4096, dtype="bf16", name="relu8-65535x4096-bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind, dtype = rng.choice(["attention", "attention", "norm", "relu8"]), rng.choice(["f32", "bf16"])
        if kind == "norm":
            c = _norm(_log_int(rng, 1, 100000), _log_int(rng, 8, 4096), dtype, rng.random() < 0.7, rng.random() < 0.8)
            if c["rows"] * c["cols"] <= 65535 * 1024:
                return c
            continue
        if kind == "relu8":
            c = _relu8(_log_int(rng, 1, 100000), _log_int(rng, 8, 8192), dtype)
            if c["rows"] * c["cols"] <= 65535 * 4096:
                return c
            continue
        heads, d = rng.choice([(8, 64), (16, 64)] if dtype == "bf16" else [(4, 64), (8, 64), (16, 64)])
        if rng.random() < 0.25:
            heads, d = rng.choice([(6, 50), (8, 40), (12, 64)])
        graph, cap = rng.choice(["bpt", "bpt", "window", "memory"]), rng.choice([0.0, 15.0, 30.0, 50.0])
        opts = dict(heads=heads, d=d, dtype=dtype, cap=cap, distance=cap == 0.0 or rng.random() < 0.6, backward=rng.random() < 0.7)
        if graph == "bpt":
            c = _attention("bpt", _log_int(rng, 32, 32768), _log_int(rng, 1, 32), **opts)
        elif graph == "window":
            c = _attention("window", _log_int(rng, 64, 16384), _log_int(rng, 16, 256), **opts)
        else:
            c = _attention("memory", _log_int(rng, 1, 8192), _log_int(rng, 1, 256), **opts)
        n_q, n_k, n_edges = _sizes(c)
        most = 3.3e9 * (1.0 if dtype == "bf16" else 0.4) * (1.0 if d == 64 else 0.25)
        if max(n_edges, 16 * max(n_q, n_k)) * heads * d <= most:
            return c


def _levels(length):
    """Nodes of every level of the binary partition of `length` tokens, and the number of each level's first node."""
    sizes = [length]
    while sizes[-1] >= 2:
        sizes.append((sizes[-1] + 1) // 2)
    return sizes, [sum(sizes[:j]) for j in range(len(sizes))]


def _edges(case, device):
    """(sources, destinations, positions of the destinations, of the sources, rows of either side)"""
    length, k = case["length"], case["k"]
    tok = torch.arange(length, device=device)
    src, dst = [], []
    if case["graph"] == "memory":
        keys, queries = tok, torch.arange(k, device=device)
        return keys.repeat(k), queries.repeat_interleave(length), (length + queries).float(), keys.float(), k, length
    if case["graph"] == "window":
        for back in range(min(length, k + 1)):
            src.append(tok[:length - back])
            dst.append(tok[back:])
        return torch.cat(src), torch.cat(dst), tok.float(), tok.float(), length, length
    sizes, first = _levels(length)
    left, child = tok - 1, torch.zeros(length, dtype=torch.bool, device=device)
    for j, start in enumerate(first):
        for _ in range(k):
            there = left >= 0                           # (a node whose sibling has been taken is met a level below, as the child itself)
            node = torch.where(child, first[max(j, 1) - 1] + 2 * left, start + left)
            src.append(node[there])
            dst.append(tok[there])
            child &= ~there
            left = left - 1
        child |= (left & 1) == 0
        left = left >> 1
        src.append(tok)
        dst.append(start + (tok >> j))
    last = [torch.clamp(((torch.arange(n, device=device) + 1) << j) - 1, max=length - 1) for j, n in enumerate(sizes)]
    pos, n = torch.cat(last).float(), sum(sizes)
    return torch.cat(src), torch.cat(dst), pos, pos, n, n


def _sizes(case):
    """(query rows, key rows, edges)"""
    length, k = case["length"], case["k"]
    if case["graph"] == "memory":
        return k, length, k * length
    if case["graph"] == "window":
        reach = min(length, k + 1)
        return length, length, reach * length - reach * (reach - 1) // 2
    src, _, _, _, n, _ = _edges(case, "cpu")
    return n, n, src.numel()


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rand = lambda shape, s=1.0: (torch.randn(shape, generator=gen, device=dev) * s).to(dtype)
    if case["op"] == "attention":
        src, dst, pos_q, pos_k, n_q, n_k = _edges(case, dev)
        h, d = case["heads"], case["d"]
        x = dict(src=src, dst=dst, pos_q=pos_q, pos_k=pos_k, q=rand((n_q, h, d)), k=rand((n_k, h, d)), v=rand((n_k, h, d)))
        if case["distance"]:
            start = 2.0 ** (-8.0 * torch.arange(1, h + 1, device=dev) / h)
            x["slopes"] = start * (1 + 0.1 * torch.randn(h, generator=gen, device=dev))
        if case["backward"]:
            x["do"] = rand((n_q, h, d), 1 / 8)
        return x
    shape = (case["rows"], case["cols"])
    if case["op"] == "norm":
        x = dict(x=rand(shape, 0.5), weight=(1 + 0.1 * torch.randn(case["cols"], generator=gen, device=dev)).to(dtype), bias=rand(case["cols"], 0.1))
        if case["residual"]:
            x["residual"] = rand(shape)
    else:
        spread = torch.exp(0.5 * torch.randn(case["cols"], generator=gen, device=dev))
        x = dict(a=(torch.randn(shape, generator=gen, device=dev) * spread).to(dtype))
    if case["op"] == "relu8" or case["backward"]:
        x["dy"] = rand(shape, 1 / 8)
    return x


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own and case["op"] == "attention":
        from bpt_amd import graphbuilder as gb
        src, dst = state.pop("src"), state.pop("dst")
        n_q, n_k = state["q"].size(0), state["k"].size(0)
        if n_q == n_k:
            csr = gb.get_csrs_device(src, dst, n_q)
        else:
            csr = gb.get_csrs_bipartite(src.cpu().numpy(), dst.cpu().numpy(), n_k, n_q)
        out_csr, in_csr, row, indptr_r, col, indptr_c = csr
        state["graph"] = tuple(t.cuda() for t in (row, indptr_r, out_csr[2], out_csr[1], col, indptr_c, in_csr[2], in_csr[1]))
    if own and case.get("backward"):
        for name in ("q", "k", "v", "slopes", "x", "residual", "weight", "bias"):
            if name in state:
                state[name].requires_grad_(True)
    return state


def run(state):
    plain, kernels = {"attention": (_plain_attention, _own_attention), "norm": (_plain_norm, _own_norm),
                      "relu8": (_plain_relu8, _own_relu8)}[state["case"]["op"]]
    return kernels(state) if own else plain(state)


# ---- through the framework ----------------------------------------------------------------------------------------------------
def _own_attention(s):
    from bpt_amd import op
    case = s["case"]
    opts = dict(score_cap=case["cap"]) if case["cap"] else {}
    if case["distance"]:
        opts.update(slopes=s["slopes"], pos=(s["pos_q"], s["pos_k"]) if case["graph"] == "memory" else s["pos_q"])
    with torch.set_grad_enabled(case["backward"]):
        o = op.bpt_attention(*s["graph"], s["q"], s["k"], s["v"], **opts)
    if not case["backward"]:
        return {"o": o}
    names = ("q", "k", "v") + (("slopes",) if case["distance"] else ())
    grads = torch.autograd.grad(o, [s[n] for n in names], s["do"])
    return dict({"o": o.detach()}, **{"d" + n: g for n, g in zip(names, grads)})


def _own_norm(s):
    from bpt_amd import op
    case = s["case"]
    with torch.set_grad_enabled(case["backward"]):
        y = op.add_layer_norm(s["x"], s.get("residual"), s["weight"], s["bias"], 1e-5)
    if not case["backward"]:
        return {"y": y}
    names = ("x",) + (("residual",) if case["residual"] else ()) + ("weight", "bias")
    grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return dict({"y": y.detach()}, **{"d" + n: g for n, g in zip(names, grads)})


def _own_relu8(s):
    from bpt_amd import graphop
    y, codes, exps = graphop.relu8_forward(s["a"])
    da, y8 = graphop.relu8_backward(s["dy"], codes, exps)
    return {"y": y, "da": da, "y8": y8}


# ---- in elementary operations, 32 bits ---------------------------------------------------------------------------------------
def _plain_attention(s):
    case = s["case"]
    q, k, v, src, dst = s["q"], s["k"], s["v"], s["src"], s["dst"]
    n_q, h, d = q.shape
    scale, cap = 1.0 / math.sqrt(d), case["cap"]
    far = (s["pos_q"][dst] - s["pos_k"][src]).abs() if case["distance"] else None
    out = {"o": torch.empty_like(q)}
    if case["backward"]:
        out.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
        if far is not None:
            out["dslopes"] = torch.empty_like(s["slopes"])
    # as many heads at a time as make tensors of at most 2 GiB of an edge's columns
    step = max(1, min(h, (1 << 29) // max(1, src.numel() * d)))
    for a in range(0, h, step):
        b = min(h, a + step)
        qe, ke, ve = q[:, a:b].float()[dst], k[:, a:b].float()[src], v[:, a:b].float()[src]
        u = (qe * ke).sum(-1) * scale
        t = torch.tanh(u / cap) if cap else None
        score = cap * t if cap else u
        if far is not None:
            score = score - s["slopes"][a:b] * far[:, None]
        rows = dst[:, None].expand(-1, b - a)
        top = torch.full((n_q, b - a), -1e9, device=q.device).scatter_reduce(0, rows, score, "amax")
        e = torch.exp(score - top[dst])
        p = e / torch.zeros((n_q, b - a), device=q.device).index_add(0, dst, e)[dst]
        out["o"][:, a:b] = torch.zeros((n_q, b - a, d), device=q.device).index_add(0, dst, p[..., None] * ve).to(q.dtype)
        if not case["backward"]:
            continue
        doe = s["do"][:, a:b].float()[dst]
        dp = (doe * ve).sum(-1)
        delta = torch.zeros((n_q, b - a), device=q.device).index_add(0, dst, p * dp)
        ds = p * (dp - delta[dst])
        if far is not None:
            out["dslopes"][a:b] = -(ds.double() * far[:, None]).sum(0).float()
        du = ds * scale
        if cap:
            du = du * (1 - t * t)
        for name, to, w, x, n in (("dq", dst, du, ke, n_q), ("dk", src, du, qe, k.size(0)), ("dv", src, p, doe, k.size(0))):
            out[name][:, a:b] = torch.zeros((n, b - a, d), device=q.device).index_add(0, to, w[..., None] * x).to(q.dtype)
    return out


def _plain_norm(s):
    case = s["case"]
    z = s["x"].float()
    if case["residual"]:
        z = z + s["residual"].float()
    w, b = s["weight"].float(), s["bias"].float()
    c = z - z.mean(1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
    xhat = c * rstd
    out = {"y": (xhat * w + b).to(s["x"].dtype)}
    if not case["backward"]:
        return out
    dy = s["dy"].float()
    g = dy * w
    dz = (rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))).to(s["x"].dtype)
    out["dx"] = dz
    if case["residual"]:
        out["dresidual"] = dz
    out["dweight"] = (dy * xhat).sum(0).to(s["x"].dtype)
    out["dbias"] = dy.sum(0).to(s["x"].dtype)
    return out


def _plain_relu8(s):
    a = s["a"]
    y = torch.relu(a)
    flat = y.float().reshape(-1)
    n = flat.numel()
    blocks = torch.nn.functional.pad(flat, (0, -n % BLOCK)).view(-1, BLOCK)
    # the smallest power of two with 255 steps up to the block's largest: m 2^e is within (255 / 256) 2^e = 255 2^(e - 8) or not
    m, e = torch.frexp(blocks.amax(1, keepdim=True))
    e = torch.where(m <= 255 / 256, e - 8, e - 7).clamp(min=-126)
    codes = torch.maximum(torch.round(torch.ldexp(blocks, -e)), (blocks > 0).float())
    y8 = torch.ldexp(codes, e).view(-1)[:n].view_as(a).to(a.dtype)
    return {"y": y, "da": torch.where(a > 0, s["dy"], torch.zeros_like(a)), "y8": y8}


# ---- from the definitions, 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, x)
    if case["op"] == "relu8":
        return _exact_relu8(x)
    wide = {n: t.double() for n, t in x.items() if n not in ("src", "dst")}
    src, dst = x["src"], x["dst"]
    n_q, h, d = x["q"].shape
    got = {n: [] for n in ("o", "dq", "dk", "dv", "dslopes")}
    for head in range(h):                               # autograd of a softmax written as exp(s) / sum exp(s), shifted by the row's largest
        leaves = [wide[n][:, head].contiguous().requires_grad_(True) for n in ("q", "k", "v")]
        u = (leaves[0].index_select(0, dst) * leaves[1].index_select(0, src)).sum(1) / d ** 0.5
        if case["cap"]:
            u = case["cap"] * torch.tanh(u / case["cap"])
        if case["distance"]:
            leaves.append(wide["slopes"][head].clone().requires_grad_(True))
            u = u - leaves[3] * (wide["pos_q"][dst] - wide["pos_k"][src]).abs()
        with torch.no_grad():
            top = torch.full((n_q,), float("-inf"), dtype=torch.float64, device=u.device).scatter_reduce(0, dst, u, "amax")
        w = torch.exp(u - top.index_select(0, dst))
        total = torch.zeros(n_q, dtype=torch.float64, device=u.device).index_add(0, dst, w)
        o = torch.zeros((n_q, d), dtype=torch.float64, device=u.device).index_add(0, dst, w[:, None] * leaves[2].index_select(0, src)) / total[:, None]
        got["o"].append(o.detach())
        if case["backward"]:
            for n, g in zip(("dq", "dk", "dv", "dslopes"), torch.autograd.grad(o, leaves, wide["do"][:, head].contiguous())):
                got[n].append(g)
    return {n: torch.stack(ts, 0 if n == "dslopes" else 1) for n, ts in got.items() if ts}


def _exact_norm(case, x):
    names = ["x"] + (["residual"] if case["residual"] else []) + ["weight", "bias"]
    leaves = {n: x[n].double().requires_grad_(True) for n in names}
    z = leaves["x"] + leaves["residual"] if case["residual"] else leaves["x"]
    y = (z - z.mean(1, keepdim=True)) / torch.sqrt(z.var(1, unbiased=False, keepdim=True) + 1e-5) * leaves["weight"] + leaves["bias"]
    out = {"y": y.detach()}
    if case["backward"]:
        out.update(zip(("d" + n for n in names), torch.autograd.grad(y, list(leaves.values()), x["dy"].double())))
    return out


def _exact_relu8(x):
    a, dy = x["a"].double(), x["dy"].double()
    y = a.clamp(min=0)
    n = y.numel()
    groups = torch.cat([y.view(-1), y.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
    top = groups.max(1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 9        # at least one too small: raised until 255 steps reach
    for _ in range(4):
        e = torch.where(255 * torch.exp2(e) < top, e + 1, e)
    step = torch.exp2(torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-126))
    y8 = torch.where(groups > 0, (groups / step).round().clamp(min=1), torch.zeros_like(groups)) * step
    return {"y": y, "da": dy * (a > 0), "y8": y8.view(-1)[:n].view_as(a)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    """Every input once and every output once.  Attention: the graph as 32-bit indices of the sides in use, two products of an edge's columns
    in the forward and four in the backward; relu8: the kept codes and exponents written and read."""
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "attention":
        n_q, n_k, n_edges = _sizes(case)
        cols, sides = case["heads"] * case["d"], 2 if case["backward"] else 1
        moved = sides * (2 * (n_q + n_k) * cols * size + 4 * (n_edges + n_q + 1))
        if case["distance"]:
            moved += 4 * (n_q + n_k) + 4 * case["heads"] * sides
        return {"bytes": moved, "flops": (12 if case["backward"] else 4) * n_edges * cols}
    n, cols = case["rows"] * case["cols"], case["cols"]
    if case["op"] == "norm":
        ins = 2 if case["residual"] else 1
        if not case["backward"]:
            return {"bytes": (n * (ins + 1) + 2 * cols) * size, "flops": n * (7 + ins)}
        return {"bytes": (n * (ins + 3) + 4 * cols) * size, "flops": n * (20 + ins)}
    return {"bytes": n * (5 * size + 2) + 2 * (n // BLOCK + 1), "flops": 8 * n}
