"""BPTBlock / BPTMemBlock with capped scores, distance and 8-bit activations together, as a training step uses them, against a float64 restatement on
the CPU; and what the blocks do without the options, on the layer norm kernel.

Tolerances: those of the blocks' other tests (2e-4 / 2e-5 for outputs, 1e-3 / 1e-4 for gradients).  The gradient of the feed-forward's second weight is
formed with activations that are off by half a step, 2^-8 of the largest of their 64 (or less than a step, where smaller than half of one):
|dO|^T (2^-8 of the block's largest) more."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def attention64(src, dst, q, k, v, cap=None, slopes=None, pos=None, table=None, etype=None):
    """(n_q, h, d) in 64 bits by gathers."""
    u = (q[dst] * (k[src] if table is None else k[src] + table[etype][:, None])).sum(-1) / math.sqrt(q.shape[-1])
    s = u if cap is None else cap * torch.tanh(u / cap)
    if slopes is not None:
        s = s - slopes * (pos[dst] - pos[src]).abs()[:, None]
    idx = dst[:, None].expand_as(s)
    top = torch.full((q.shape[0], q.shape[1]), -1e300, dtype=s.dtype).scatter_reduce(0, idx, s.detach(), "amax")
    w = torch.exp(s - top[dst])
    total = torch.zeros_like(top).index_add(0, dst, w)
    return torch.zeros_like(q).index_add(0, dst, (w / total[dst])[..., None] * v[src])


def to_dev(csr):
    return tuple(tuple(t.to(DEV) for t in c) if isinstance(c, (tuple, list)) else c.to(DEV) for c in csr)


def close(a, b, what, rtol, atol, more=0.0):
    a, b = a.detach().cpu().double(), b.detach()
    excess = (a - b).abs() - atol - rtol * b.abs() - more
    assert excess.max() <= 0, f"{what}: beyond by {excess.max():.3e}, largest error {(a - b).abs().max():.3e}"


def case(L=300, seed=1, dim=512):
    from bpt_amd import graphbuilder as gb
    g = gb.BinaryPartition(L, True, 2, 10)
    src, dst, etype = g.get_edges()
    n = g.number_of_nodes
    gen = torch.Generator().manual_seed(seed)
    return dict(src=torch.from_numpy(src), dst=torch.from_numpy(dst), etype=torch.from_numpy(etype.astype(np.int64)), n=n, csr=gb.get_csrs(src, dst, n),
                pos=torch.from_numpy(g.get_pos()).float(), h=torch.randn(n, dim, generator=gen), gout=torch.randn(n, dim, generator=gen))


@pytest.mark.parametrize("rel_pos", [False, True])
@pytest.mark.parametrize("dims", [(512, 8, 256), (300, 6, 128), (96, 3, 64), (160, 2, 64)], ids=str)      # fused, narrow, padded, the chain (80 columns)
def test_block_with_all_options(dims, rel_pos):
    from bpt_amd.block import BPTBlock
    dim, heads, ff = dims
    c = case(dim=dim)
    torch.manual_seed(7)
    blk = BPTBlock(dim, heads, ff, rel_pos=rel_pos, drop_h=0.0, drop_a=0.0, score_cap=5.0, distance=True, keep8=True)
    blk.reset_parameters()
    ref = copy.deepcopy(blk).double()
    blk = blk.to(DEV)
    h = c["h"].to(DEV).requires_grad_(True)
    out = blk(h, to_dev(c["csr"]), c["etype"].to(DEV) if rel_pos else None, c["pos"].to(DEV))
    out.backward(c["gout"].to(DEV))

    h64 = c["h"].double().requires_grad_(True)
    split = lambda proj: proj(h64).view(-1, heads, dim // heads)
    a = attention64(c["src"], c["dst"], split(ref.proj_q), split(ref.proj_k), split(ref.proj_v), 5.0, ref.slopes, c["pos"].double(),
                    ref.embed_ak.weight if rel_pos else None, c["etype"])
    x = ref.norm_in(h64 + ref.proj_o(a.reshape(-1, dim)))
    act = torch.relu(ref.ffn[0].w_1(x))
    act.retain_grad()
    f = ref.ffn[0].w_2(act)
    f.retain_grad()
    out64 = ref.norm_inter(x + f)
    out64.backward(c["gout"].double())
    close(out, out64, "block output", 2e-4, 2e-5)
    close(h.grad, h64.grad, "d input", 1e-3, 1e-4)
    blocks = torch.nn.functional.pad(act.detach().reshape(-1), (0, -act.numel() % 64)).view(-1, 64).amax(1).repeat_interleave(64)[:act.numel()].view_as(act)
    eight = f.grad.abs().t() @ (blocks * 2.0 ** -8)
    for (name, p), (_, pr) in zip(blk.named_parameters(), ref.named_parameters()):
        close(p.grad, pr.grad, f"d {name}", 1e-3, 1e-4, eight if name == "ffn.0.w_2.weight" else 0.0)


def test_mem_block_with_options():
    from bpt_amd import graphbuilder as gb
    from bpt_amd.block import BPTMemBlock
    enc, dec = [gb.BinaryPartition(n, False, 2, 10) for n in (40, 30)], [gb.BinaryPartition(n, True, 2, 10) for n in (25, 60)]
    src, dst, _, pos, n = gb.merge_graphs(dec)
    isrc, idst, n_mem, n_dec = gb.inter_graph_edges(enc, dec)
    torch.manual_seed(5)
    blk = BPTMemBlock(512, 8, 256, drop_h=0.0, drop_a=0.0, score_cap=4.0, distance=True, keep8=True)
    blk.reset_parameters()
    ref = copy.deepcopy(blk).double()
    blk = blk.to(DEV)
    gen = torch.Generator().manual_seed(2)
    h0, mem0, gout = (torch.randn(m, 512, generator=gen) for m in (n_dec, n_mem, n_dec))
    h, mem, pos = h0.to(DEV).requires_grad_(True), mem0.to(DEV).requires_grad_(True), torch.from_numpy(pos).float()
    out = blk(h, to_dev(gb.get_csrs(src, dst, n)), mem, to_dev(gb.get_csrs_bipartite(isrc, idst, n_mem, n_dec)), pos=pos.to(DEV))
    out.backward(gout.to(DEV))
    t = torch.from_numpy
    h64, mem64 = h0.double().requires_grad_(True), mem0.double().requires_grad_(True)
    split = lambda proj, x: proj(x).view(-1, 8, 64)
    a = attention64(t(src), t(dst), split(ref.proj_q[0], h64), split(ref.proj_k[0], h64), split(ref.proj_v[0], h64), 4.0, ref.slopes, pos.double())
    x = ref.norm_in[0](h64 + ref.proj_o[0](a.reshape(-1, 512)))
    a = attention64(t(isrc), t(idst), split(ref.proj_q[1], x), split(ref.proj_k[1], mem64), split(ref.proj_v[1], mem64), 4.0)
    x = ref.norm_in[1](x + ref.proj_o[1](a.reshape(-1, 512)))
    out64 = ref.norm_inter(x + ref.ffn[0].w_2(torch.relu(ref.ffn[0].w_1(x))))
    out64.backward(gout.double())
    close(out, out64, "block output", 2e-4, 2e-5)
    close(h.grad, h64.grad, "d input", 1e-3, 1e-4)
    close(mem.grad, mem64.grad, "d memory", 1e-3, 1e-4)
    for (name, p), (_, pr) in zip(blk.named_parameters(), ref.named_parameters()):
        if name != "ffn.0.w_2.weight":
            close(p.grad, pr.grad, f"d {name}", 1e-3, 1e-4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step_with_dropout_repeats(dtype):
    """All options and all dropouts: the same seeds give the same bits, and every parameter has a finite gradient."""
    from bpt_amd.block import BPTBlock
    c = case(500)
    torch.manual_seed(3)
    blk = BPTBlock(512, 8, 1024, rel_pos=True, drop_h=0.1, drop_a=0.1, score_cap=10.0, distance=True, keep8=True).to(DEV).to(dtype)
    csr, h, pos = to_dev(c["csr"]), c["h"].to(DEV).to(dtype), c["pos"].to(DEV)
    runs = []
    for _ in range(2):
        torch.manual_seed(11)
        blk.zero_grad()
        out = blk(h, csr, c["etype"].to(DEV), pos)
        out.backward(c["gout"].to(DEV).to(dtype))
        runs.append([out.detach()] + [p.grad.clone() for p in blk.parameters()])
        assert all(torch.isfinite(x.float()).all() and x.abs().max() > 0 for x in runs[-1])
    assert torch.equal(runs[0][0], runs[1][0])


def test_keep8_keeps_less():
    from bpt_amd.block import PositionwiseFeedForward
    x = torch.randn(4096, 512, device=DEV, requires_grad=True)
    held = []
    for keep8 in (False, True):
        f = PositionwiseFeedForward(512, 2048, 0.1, keep8=keep8).to(DEV)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = f(x)
        held.append(torch.cuda.memory_allocated() - before - out.numel() * 4)
        del out
    assert held[1] <= 4096 * 2048 * (1 + 1 / 64) + 2 ** 20 and held[0] >= 8 * 4096 * 2048


def test_keep8_calls_modules_that_are_not_as_they_were():
    """A hook on the second layer, a layer of another class and a dropout of everything: torch's modules run, with their results."""
    from bpt_amd.block import PositionwiseFeedForward
    x = torch.randn(50, 64, device=DEV)

    class Doubled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    def pair(p=0.0):
        torch.manual_seed(3)
        plain = PositionwiseFeedForward(64, 256, p).to(DEV)
        kept = copy.deepcopy(plain)
        kept.keep8 = True
        return plain, kept
    plain, kept = pair()
    for f in (plain, kept):
        f.w_2.register_forward_hook(lambda m, i, o: 3 * o)
    assert torch.equal(plain(x), kept(x))
    plain, kept = pair()
    for f in (plain, kept):
        f.w_2.__class__ = Doubled
    assert torch.equal(plain(x), kept(x))
    plain, kept = pair(1.0)
    assert torch.equal(plain(x), kept(x)) and torch.equal(kept(x), kept.w_2.bias.expand(50, 64))
    plain, kept = pair()
    assert torch.equal(plain.cpu()(x.cpu()), kept.cpu()(x.cpu()))


def test_the_norms_of_a_block_are_layer_norms():
    """The kernel and the module agree to rounding; a hook on the module, a module of the caller's and autocast are honoured."""
    from bpt_amd.block import BPTBlock
    c = case(200)
    csr, h = to_dev(c["csr"]), c["h"].to(DEV)
    torch.manual_seed(1)
    blk = BPTBlock(512, 8, 256, drop_h=0.0, drop_a=0.0).to(DEV)
    out = blk(h, csr)
    seen = []
    handle = blk.norm_in.register_forward_hook(lambda m, i, o: seen.append(o))
    assert (blk(h, csr) - out).abs().max() < 1e-5 and len(seen) == 1
    handle.remove()
    blk(h, csr)
    assert len(seen) == 1
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert blk(h, csr).dtype == torch.float32
    blk.norm_inter = torch.nn.Identity()
    assert (blk(h, csr) - out).abs().max() > 0.1


def test_blocks_without_the_options_are_as_they_were():
    from bpt_amd.block import BPTBlock, PositionwiseFeedForward
    blk = BPTBlock(64, 2, 32)
    state = pickle.loads(pickle.dumps(blk))
    for m in state.modules():                                     # as one pickled before there were options
        for name in ("score_cap", "distance", "keep8"):
            m.__dict__.pop(name, None)
    c = case(30, dim=64)
    torch.manual_seed(0)
    assert torch.isfinite(state.to(DEV).eval()(c["h"].to(DEV), to_dev(c["csr"]))).all()
    assert "slopes" not in dict(blk.named_parameters()) and not PositionwiseFeedForward(8, 8).keep8
    with pytest.raises(ValueError, match="pos"):
        BPTBlock(64, 2, 32, distance=True).to(DEV)(c["h"].to(DEV), to_dev(c["csr"]))
