"""What the operators that a block runs beside its attention kernels, and the bias it adds to their scores, are measured on: passes through
the public entry points, and the same passes in elementary torch operations.

A case is a dict of plain values; `op` names the operator:

  "linear"     op.linear_act: residual + dropout(act(x weight^T + bias)) of `rows` rows, `inner` columns in and `outer` out; `act` "none", "relu" or
               "gelu" (with the error function); `bias`, `residual`: with them; `dropout`: share dropped
  "dropout"    op.dropout of `rows` x `cols` elements; `residual`: the result is added to another tensor
  "attention"  op.bpt_attention with a learned bias of every edge's bucket and head added to the scaled score, bias_table[bucket, head].  `graph`: "bpt" a
               causal binary-partition graph of `length` tokens, `k` neighbours per level; "window" every token attends to the `k` tokens before
               it and itself; "memory" `k` query rows that attend to all of `length` key rows.  `heads`, `d`, `buckets`: half of them hold one
               distance of the positions each, the others widen by a constant factor, as such models have them

`dtype` "f32" or "bf16"; `backward`: with the gradients of everything that has one.

Node features are N(0, 1), as projections of layer-normalised states are, incoming gradients N(0, 1) / 8, weights N(0, 1 / inner).  Where relu decides, x and
weight are rounded to steps that make every sum exact in 32 bits, and the bias lies half a step off, so that which activations are positive does
not hang on the order of a sum.  Dropout's decisions are Philox-4x32-10 words (Salmon et al. 2011) of the seed and the element's place in memory: element i
takes word i % 4 of counter (i // 4, 0) under the seed's two halves, and is dropped where the word is below share * 2^32.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
MOST = 6.0e11           # operations of a product of the largest listed case, no drawn case has more


def _linear(rows, inner, outer, act="none", bias=True, residual=False, dropout=0.0, dtype="f32", backward=True, name=None):
    c = dict(op="linear", rows=rows, inner=inner, outer=outer, act=act, bias=bias, residual=residual, dropout=dropout, dtype=dtype, backward=backward)
    return c if name is None else dict(c, name=name)


def _dropout(rows, cols, share=0.1, residual=False, dtype="f32", name=None):
    c = dict(op="dropout", rows=rows, cols=cols, dropout=share, residual=residual, dtype=dtype, backward=True)
    return c if name is None else dict(c, name=name)


def _attention(graph, length, k, heads=8, d=64, buckets=32, dtype="f32", backward=True, name=None):
    c = dict(op="attention", graph=graph, length=length, k=k, heads=heads, d=d, buckets=buckets, dtype=dtype, backward=backward)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a decoder that takes one new token: the first layer of its feed-forward
        _linear(1, 512, 2048, act="relu", backward=False, name="linear-1x512-2048-relu-f32"),
        # 48 hypotheses side by side: what attention gives, projected and added to the states
        _linear(48, 512, 512, bias=False, residual=True, dtype="bf16", backward=False, name="linear-48x512-512-res-bf16"),
        # a classification batch of 6 heads x 50 columns: rows that do not start on 16 bytes
        _linear(33598, 300, 600, act="gelu", dtype="bf16", name="linear-33598x300-600-gelu-bf16"),
        # the first layer of the feed-forward in training, 8192 tokens of context
        _linear(16383, 512, 2048, act="relu", dropout=0.1, name="linear-16383x512-2048-relu-drop-f32"),
        # the second layer, its dropout and the residual sum, 32768 tokens: the largest product
        _linear(65535, 4096, 1024, residual=True, dropout=0.1, dtype="bf16", name="linear-65535x4096-1024-res-drop-bf16"),
        # one short sentence's states
        _dropout(127, 300, name="dropout-127x300-f32"),
        # those of 8192 tokens, added to the residual stream
        _dropout(16383, 512, residual=True, name="dropout-16383x512-res-f32"),
        # those of 32768 tokens
        _dropout(65535, 1024, share=0.3, dtype="bf16", name="dropout-65535x1024-bf16"),
        # a decoder's one new token, its row attends to a memory of 2048 nodes
        _attention("memory", 2048, 1, backward=False, name="bias-row2048-f32"),
        # one paragraph-sized sequence in training
        _attention("bpt", 512, 4, name="bias-L512-f32"),
        # a character-level language model's layer, 8192 tokens of context
        _attention("bpt", 8192, 4, name="bias-L8192-f32"),
        # long context, wide neighbourhood, 16 heads
        _attention("bpt", 32768, 8, heads=16, buckets=64, dtype="bf16", name="bias-L32768-k8-bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind, dtype = rng.choice(["linear", "linear", "attention", "dropout"]), rng.choice(["f32", "bf16"])
        if kind == "linear":
            c = _linear(_log_int(rng, 1, 65535), _log_int(rng, 16, 4096), _log_int(rng, 16, 4096), rng.choice(["none", "relu", "gelu"]), rng.random() < 0.7,
                        rng.random() < 0.4, rng.choice([0.0, 0.1, 0.3]), dtype, rng.random() < 0.7)
            if rng.random() < 0.6:                      # widths of whole vectors, as models have them
                c["inner"], c["outer"] = (max(16, -(-c[n] // 16) * 16) for n in ("inner", "outer"))
            if 2.0 * c["rows"] * c["inner"] * c["outer"] <= MOST * (1.0 if dtype == "bf16" else 0.15):
                return c
            continue
        if kind == "dropout":
            c = _dropout(_log_int(rng, 1, 100000), _log_int(rng, 8, 4096), rng.choice([0.1, 0.2, 0.5]), rng.random() < 0.5, dtype)
            if c["rows"] * c["cols"] <= 65535 * 1024:
                return c
            continue
        heads, d = rng.choice([(8, 64), (16, 64)] if dtype == "bf16" else [(4, 64), (8, 64), (16, 64)])
        if rng.random() < 0.25:
            heads, d = rng.choice([(6, 50), (8, 40), (12, 64)])
        graph = rng.choice(["bpt", "bpt", "window", "memory"])
        opts = dict(heads=heads, d=d, buckets=2 * rng.randint(4, 48), dtype=dtype, backward=rng.random() < 0.7)
        if graph == "bpt":
            c = _attention("bpt", _log_int(rng, 32, 32768), _log_int(rng, 1, 32), **opts)
        elif graph == "window":
            c = _attention("window", _log_int(rng, 64, 16384), _log_int(rng, 16, 256), **opts)
        else:
            c = _attention("memory", _log_int(rng, 64, 8192), _log_int(rng, 1, 256), **opts)
        n_q, n_k, n_edges = _sizes(c)
        most = 3.3e9 * (1.0 if dtype == "bf16" else 0.4) * (1.0 if d == 64 else 0.25)
        if max(n_edges, 16 * max(n_q, n_k)) * heads * d <= most:
            return c


# ---- graphs and buckets --------------------------------------------------------------------------------------------------------
def _levels(length):
    """Nodes of every level of the binary partition of `length` tokens, and the number of each level's first node."""
    sizes = [length]
    while sizes[-1] >= 2:
        sizes.append((sizes[-1] + 1) // 2)
    return sizes, [sum(sizes[:j]) for j in range(len(sizes))]


def _edges(case, device):
    """(sources, destinations, distances of their positions, rows of either side)"""
    length, k = case["length"], case["k"]
    tok = torch.arange(length, device=device)
    src, dst = [], []
    if case["graph"] == "memory":
        queries = torch.arange(k, device=device)
        src, dst = tok.repeat(k), queries.repeat_interleave(length)
        return src, dst, length + dst - src, k, length
    if case["graph"] == "window":
        for back in range(min(length, k + 1)):
            src.append(tok[:length - back])
            dst.append(tok[back:])
        src, dst = torch.cat(src), torch.cat(dst)
        return src, dst, dst - src, length, length
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
    pos, src, dst, n = torch.cat(last), torch.cat(src), torch.cat(dst), sum(sizes)
    return src, dst, (pos[dst] - pos[src]).abs(), n, n


def _buckets(far, n):
    """Buckets of distances: one each below n / 2, then widening by a constant factor up to 8192."""
    half = n // 2
    borders = [round(half * (8192.0 / half) ** (i / half)) for i in range(1, half)]
    return torch.where(far < half, far, half + torch.bucketize(far, torch.tensor(borders, device=far.device), right=True)).clamp(max=n - 1)


def _sizes(case):
    """(query rows, key rows, edges)"""
    length, k = case["length"], case["k"]
    if case["graph"] == "memory":
        return k, length, k * length
    if case["graph"] == "window":
        reach = min(length, k + 1)
        return length, length, reach * length - reach * (reach - 1) // 2
    src, _, _, n, _ = _edges(case, "cpu")
    return n, n, src.numel()


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rand = lambda shape, s=1.0: (torch.randn(shape, generator=gen, device=dev) * s).to(dtype)
    if case["op"] == "attention":
        src, dst, far, n_q, n_k = _edges(case, dev)
        h, d = case["heads"], case["d"]
        x = dict(src=src, dst=dst, buckets=_buckets(far, case["buckets"]), q=rand((n_q, h, d)), k=rand((n_k, h, d)), v=rand((n_k, h, d)),
                 table=rand((case["buckets"], h), 0.5))
        if case["backward"]:
            x["do"] = rand((n_q, h, d), 1 / 8)
        return x
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        x = dict(x=rand(shape), dy=rand(shape, 1 / 8), seed=(seed * 0x9E3779B97F4A7C15 + 12345) % 2 ** 62)
        if case["residual"]:
            x["residual"] = rand(shape)
        return x
    rows, inner, outer = case["rows"], case["inner"], case["outer"]
    x = dict(x=rand((rows, inner)), weight=rand((outer, inner), inner ** -0.5), seed=(seed * 0x9E3779B97F4A7C15 + 54321) % 2 ** 62)
    if case["act"] == "relu":
        step = 2.0 ** (round(math.log2(inner ** -0.5)) - 4)
        x["x"] = (x["x"].float() * 8).round().clamp(-40, 40).div(8).to(dtype)
        x["weight"] = (x["weight"].float() / step).round().clamp(-80, 80).mul(step).to(dtype)
        if case["bias"]:
            x["bias"] = ((2 * torch.randint(-60, 60, (outer,), generator=gen, device=dev) + 1) * (step / 16)).to(dtype)
    elif case["bias"]:
        x["bias"] = rand((outer,), 0.1)
    if case["residual"]:
        x["residual"] = rand((rows, outer))
    if case["backward"]:
        x["dy"] = rand((rows, outer), 1 / 8)
    return x


GRADIENTS = {"linear": ("x", "weight", "bias", "residual"), "dropout": ("x", "residual"), "attention": ("q", "k", "v", "table")}


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
    if own and case["backward"]:
        for name in GRADIENTS[case["op"]]:
            if name in state:
                state[name].requires_grad_(True)
    return state


def run(state):
    plain = {"linear": _plain_linear, "dropout": _plain_dropout, "attention": _plain_attention}
    return _own(state) if own else plain[state["case"]["op"]](state)


# ---- through the framework ----------------------------------------------------------------------------------------------------
def _own(s):
    from bpt_amd import op
    case = s["case"]
    with torch.set_grad_enabled(case["backward"]):
        if case["op"] == "linear":
            y = op.linear_act(s["x"], s["weight"], s.get("bias"), activation=None if case["act"] == "none" else case["act"], residual=s.get("residual"),
                              dropout_p=case["dropout"], seed=s["seed"])
        elif case["op"] == "dropout":
            y = op.dropout(s["x"], case["dropout"], seed=s["seed"], residual=s.get("residual"))
        else:
            y = op.bpt_attention(*s["graph"], s["q"], s["k"], s["v"], bias_table=s["table"], buckets=s["buckets"])
    if not case["backward"]:
        return {"y": y}
    names = [n for n in GRADIENTS[case["op"]] if n in s]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["do"] if case["op"] == "attention" else s["dy"])
    return dict({"y": y.detach()}, **{"d" + n: g for n, g in zip(names, grads)})


# ---- in elementary operations, 32 bits ---------------------------------------------------------------------------------------
M32 = 0xFFFFFFFF


def _philox(seed, n, device):
    """n words of Philox-4x32-10, in products of 64 bits whose upper half is masked out (they wrap, the words do not)."""
    c0 = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    c1 = c0 >> 32
    c0 = c0 & M32
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & M32, seed >> 32 & M32
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (q >> 32 & M32) ^ c1 ^ k0, q & M32, (p >> 32 & M32) ^ c3 ^ k1, p & M32
        k0, k1 = k0 + 0x9E3779B9 & M32, k1 + 0xBB67AE85 & M32
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _keep(seed, share, shape, device):
    """1 / (1 - share) where an element is kept, 0 elsewhere, in 32 bits."""
    n = shape[0] * shape[1]
    return torch.where(_philox(seed, n, device) >= int(share * 2 ** 32), 1.0 / (1.0 - share), 0.0).to(torch.float32).view(shape)


def _plain_linear(s):
    case = s["case"]
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    a = x @ w.t()
    if case["bias"]:
        a = a + s["bias"].float()
    phi = 0.5 * (1 + torch.erf(a * 0.5 ** 0.5)) if case["act"] == "gelu" else None
    y = torch.clamp(a, min=0) if case["act"] == "relu" else a * phi if case["act"] == "gelu" else a
    keep = _keep(s["seed"], case["dropout"], y.shape, y.device) if case["dropout"] else None
    if keep is not None:
        y = y * keep
    if case["residual"]:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if not case["backward"]:
        return out
    g = s["dy"].float()
    if keep is not None:
        g = g * keep
    if case["act"] == "relu":
        g = torch.where(a > 0, g, torch.zeros_like(g))
    elif case["act"] == "gelu":
        g = g * (phi + a * torch.exp(-0.5 * a * a) * (2 * math.pi) ** -0.5)
    out.update(dx=(g @ w).to(dtype), dweight=(g.t() @ x).to(dtype))
    if case["bias"]:
        out["dbias"] = g.sum(0).to(dtype)
    if case["residual"]:
        out["dresidual"] = s["dy"]
    return out


def _plain_dropout(s):
    case = s["case"]
    keep = _keep(s["seed"], case["dropout"], s["x"].shape, s["x"].device)
    y = s["x"].float() * keep
    out = {"dx": (s["dy"].float() * keep).to(s["x"].dtype)}
    if case["residual"]:
        y = y + s["residual"].float()
        out["dresidual"] = s["dy"]
    return dict({"y": y.to(s["x"].dtype)}, **out)


def _plain_attention(s):
    case = s["case"]
    q, k, v, table, src, dst, buckets = s["q"], s["k"], s["v"], s["table"].float(), s["src"], s["dst"], s["buckets"]
    n_q, h, d = q.shape
    scale = 1.0 / math.sqrt(d)
    out = {"y": torch.empty_like(q)}
    if case["backward"]:
        out.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v), dtable=torch.empty_like(s["table"]))
    # as many heads at a time as make tensors of at most 2 GiB of an edge's columns
    step = max(1, min(h, (1 << 29) // max(1, src.numel() * d)))
    for a in range(0, h, step):
        b = min(h, a + step)
        qe, ke, ve = q[:, a:b].float()[dst], k[:, a:b].float()[src], v[:, a:b].float()[src]
        score = (qe * ke).sum(-1) * scale + table[:, a:b][buckets]
        rows = dst[:, None].expand(-1, b - a)
        top = torch.full((n_q, b - a), -1e9, device=q.device).scatter_reduce(0, rows, score, "amax")
        e = torch.exp(score - top[dst])
        p = e / torch.zeros((n_q, b - a), device=q.device).index_add(0, dst, e)[dst]
        out["y"][:, a:b] = torch.zeros((n_q, b - a, d), device=q.device).index_add(0, dst, p[..., None] * ve).to(q.dtype)
        if not case["backward"]:
            continue
        doe = s["do"][:, a:b].float()[dst]
        dp = (doe * ve).sum(-1)
        delta = torch.zeros((n_q, b - a), device=q.device).index_add(0, dst, p * dp)
        ds = p * (dp - delta[dst])
        # (a long sum: 64 bits)
        out["dtable"][:, a:b] = torch.zeros((case["buckets"], b - a), dtype=torch.float64, device=q.device).index_add(0, buckets, ds.double()).to(q.dtype)
        for name, to, w, x, n in (("dq", dst, ds * scale, ke, n_q), ("dk", src, ds * scale, qe, k.size(0)), ("dv", src, p, doe, k.size(0))):
            out[name][:, a:b] = torch.zeros((n, b - a, d), device=q.device).index_add(0, to, w[..., None] * x).to(q.dtype)
    return out


# ---- from the definitions, 64 bits ------------------------------------------------------------------------------------------
def _mulhilo(a, c):
    """Upper and lower words of a * c, of a tensor of words and a constant, by halves of 16 bits."""
    a0, a1, c0, c1 = a & 0xFFFF, a >> 16, c & 0xFFFF, c >> 16
    low, mid = a0 * c0, a1 * c0 + (a0 * c0 >> 16)
    mid2 = a0 * c1 + (mid & 0xFFFF)
    return a1 * c1 + (mid >> 16) + (mid2 >> 16), (mid2 & 0xFFFF) << 16 | low & 0xFFFF


def _kept(case, x, shape, device):
    """Dropout's factors in 64 bits, four words of a counter at a time."""
    n = shape[0] * shape[1]
    number = torch.arange(-(-n // 4), device=device)
    ctr, key = [number % 2 ** 32, number // 2 ** 32, torch.zeros_like(number), torch.zeros_like(number)], [x["seed"] % 2 ** 32, x["seed"] // 2 ** 32 % 2 ** 32]
    for turn in range(10):
        h0, l0 = _mulhilo(ctr[0], 0xD2511F53)
        h1, l1 = _mulhilo(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ (key[0] + turn * 0x9E3779B9) % 2 ** 32, l1, h0 ^ ctr[3] ^ (key[1] + turn * 0xBB67AE85) % 2 ** 32, l0]
    kept = torch.empty((number.numel(), 4), dtype=torch.float64, device=device)
    for word in range(4):
        kept[:, word] = (ctr[word].double() >= math.floor(case["dropout"] * 2.0 ** 32)).double() / (1.0 - case["dropout"])
    return kept.view(-1)[:n].view(shape)


def exact(case, seed):
    x = _inputs(case, seed)
    names = [n for n in GRADIENTS[case["op"]] if n in x]
    if case["op"] == "attention":
        return _exact_attention(case, x)
    leaves = {n: x[n].double().requires_grad_(case["backward"]) for n in names}
    if case["op"] == "linear":
        y = torch.matmul(leaves["x"], leaves["weight"].transpose(0, 1))
        y = y + leaves["bias"] if case["bias"] else y
        if case["act"] == "relu":
            y = (y + y.abs()) / 2
        elif case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
    else:
        y = leaves["x"]
    if case["dropout"]:
        y = y * _kept(case, x, y.shape, y.device)
    if case["residual"]:
        y = y + leaves["residual"]
    out = {"y": y.detach()}
    if case["backward"]:
        out.update(zip(("d" + n for n in names), torch.autograd.grad(y, list(leaves.values()), x["dy"].double())))
    return out


def _exact_attention(case, x):
    wide = {n: x[n].double() for n in ("q", "k", "v", "table", "do") if n in x}
    src, dst = x["src"], x["dst"]
    n_q, h, d = x["q"].shape
    got = {n: [] for n in ("y", "dq", "dk", "dv", "dtable")}
    for head in range(h):                               # autograd of a softmax written as exp(s) / sum exp(s), shifted by the row's largest
        leaves = [wide[n][:, head].contiguous().requires_grad_(True) for n in ("q", "k", "v", "table")]
        u = (leaves[0].index_select(0, dst) * leaves[1].index_select(0, src)).sum(1) / d ** 0.5 + leaves[3].index_select(0, x["buckets"])
        with torch.no_grad():
            top = torch.full((n_q,), float("-inf"), dtype=torch.float64, device=u.device).scatter_reduce(0, dst, u, "amax")
        w = torch.exp(u - top.index_select(0, dst))
        total = torch.zeros(n_q, dtype=torch.float64, device=u.device).index_add(0, dst, w)
        o = torch.zeros((n_q, d), dtype=torch.float64, device=u.device).index_add(0, dst, w[:, None] * leaves[2].index_select(0, src)) / total[:, None]
        got["y"].append(o.detach())
        if case["backward"]:
            for n, g in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(o, leaves, wide["do"][:, head].contiguous())):
                got[n].append(g)
    return {n: torch.stack(ts, 1) for n, ts in got.items() if ts}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    """Every input once and every output once.  Attention: the graph as 32-bit indices of the sides in use and the buckets as they are given, two products
    of an edge's columns in the forward and four in the backward."""
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "attention":
        n_q, n_k, n_edges = _sizes(case)
        cols, sides = case["heads"] * case["d"], 2 if case["backward"] else 1
        moved = sides * (2 * (n_q + n_k) * cols * size + 4 * (n_edges + n_q + 1) + case["buckets"] * case["heads"] * size) + 8 * n_edges
        return {"bytes": moved, "flops": (12 if case["backward"] else 4) * n_edges * cols}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size * (5 if case["residual"] else 4), "flops": 2 * n}
    x, w, y = case["rows"] * case["inner"], case["inner"] * case["outer"], case["rows"] * case["outer"]
    one = x + w + y + (y if case["residual"] else 0) + (case["outer"] if case["bias"] else 0)
    if not case["backward"]:
        return {"bytes": one * size, "flops": 2 * case["inner"] * y}
    return {"bytes": (one + x + w + y + (case["outer"] if case["bias"] else 0)) * size, "flops": 6 * case["inner"] * y}
