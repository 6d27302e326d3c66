"""BPTBlock and BPTMemBlock with epilogue and bucket_bias: the operators together, as a layer runs them."""
import copy
import math

import pytest
import torch

import philox_model
from test_gpu_block_options import case, close, to_dev

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def attention64(src, dst, q, k, v, table=None, buckets=None):
    n, heads, d = q.shape
    s = (q[dst] * k[src]).sum(-1) / math.sqrt(d)
    if table is not None:
        s = s + torch.where((buckets < table.size(0))[:, None], table[buckets.clamp(max=table.size(0) - 1)], 0.0)
    idx = dst[:, None].expand(-1, heads)
    top = torch.full((n, heads), -1e300, dtype=torch.float64).scatter_reduce(0, idx, s.detach(), "amax")
    w = torch.exp(s - top[dst])
    p = w / torch.zeros((n, heads), dtype=torch.float64).index_add(0, dst, w)[dst]
    return torch.zeros((n, heads, d), dtype=torch.float64).index_add(0, dst, p[..., None] * v[src])


def keep(seed, p, shape):
    return torch.from_numpy(philox_model.keep(seed, p, shape[0] * shape[1])).view(shape).double() / (1 - p) if p else torch.ones(shape, dtype=torch.float64)


@pytest.mark.parametrize("drop_h", [0.0, 0.2])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("dims", [(512, 8, 256), (300, 6, 130), (96, 3, 64), (160, 2, 64)], ids=str)
def test_block_against_the_formula(dims, keep8, drop_h):
    """Dropout's decisions are the generator's words of the seeds that the layer draws in turn.  Tolerances as in the tests of the other options."""
    from bpt_amd.block import BPTBlock
    if keep8 and drop_h:
        pytest.skip("relu_linear8 has decisions of its own")
    dim, heads, ff = dims
    c = case(dim=dim)
    torch.manual_seed(7)
    blk = BPTBlock(dim, heads, ff, drop_h=drop_h, drop_a=0.0, keep8=keep8, epilogue=True, bucket_bias=12)
    blk.reset_parameters()
    ref = copy.deepcopy(blk).double()
    blk = blk.to(DEV)
    h = c["h"].to(DEV).requires_grad_(True)
    torch.manual_seed(23)
    out = blk(h, to_dev(c["csr"]), c["etype"].to(DEV))
    out.backward(c["gout"].to(DEV))

    torch.manual_seed(23)
    seeds = [int(torch.randint(0, 2 ** 62, (1,)).item()) for _ in range(3)]
    n = c["n"]
    h64 = c["h"].double().requires_grad_(True)
    split = lambda proj: proj(h64).view(-1, heads, dim // heads)
    a = attention64(c["src"], c["dst"], split(ref.proj_q), split(ref.proj_k), split(ref.proj_v), ref.bias_table, c["etype"])
    x = ref.norm_in(h64 + ref.proj_o(a.reshape(-1, dim)) * keep(seeds[0], drop_h, (n, dim)))
    act = torch.relu(ref.ffn[0].w_1(x)) * keep(seeds[1], drop_h, (n, ff))
    act.retain_grad()
    f = ref.ffn[0].w_2(act)
    f.retain_grad()
    out64 = ref.norm_inter(x + f * keep(seeds[2], drop_h, (n, dim)))
    out64.backward(c["gout"].double())
    close(out, out64, "block output", 2e-4, 2e-5)
    close(h.grad, h64.grad, "d input", 1e-3, 1e-4)
    blocks = torch.nn.functional.pad(act.detach().reshape(-1), (0, -act.numel() % 64)).view(-1, 64).amax(1).repeat_interleave(64)[:act.numel()].view_as(act)
    eight = f.grad.abs().t() @ (blocks * 2.0 ** -8)
    for (name, p), (_, pr) in zip(blk.named_parameters(), ref.named_parameters()):
        close(p.grad, pr.grad, f"d {name}", 1e-3, 1e-4, eight if keep8 and name == "ffn.0.w_2.weight" else 0.0)


def test_mem_block_against_the_formula():
    from bpt_amd import graphbuilder as gb
    from bpt_amd.block import BPTMemBlock
    enc, dec = [gb.BinaryPartition(n, False, 2, 10) for n in (40, 30)], [gb.BinaryPartition(n, True, 2, 10) for n in (25, 60)]
    src, dst, etype, _, n = gb.merge_graphs(dec)
    isrc, idst, n_mem, n_dec = gb.inter_graph_edges(enc, dec)
    torch.manual_seed(5)
    blk = BPTMemBlock(512, 8, 256, drop_h=0.0, drop_a=0.0, epilogue=True, bucket_bias=50)
    blk.reset_parameters()
    ref = copy.deepcopy(blk).double()
    blk = blk.to(DEV)
    gen = torch.Generator().manual_seed(2)
    h0, mem0, gout = (torch.randn(m, 512, generator=gen) for m in (n_dec, n_mem, n_dec))
    t = lambda x: torch.as_tensor(x).long()
    h, mem = h0.to(DEV).requires_grad_(True), mem0.to(DEV).requires_grad_(True)
    out = blk(h, to_dev(gb.get_csrs(src, dst, n)), mem, to_dev(gb.get_csrs_bipartite(isrc, idst, n_mem, n_dec)), t(etype).to(DEV))
    out.backward(gout.to(DEV))
    h64, mem64 = h0.double().requires_grad_(True), mem0.double().requires_grad_(True)
    split = lambda proj, x: proj(x).view(-1, 8, 64)
    a = attention64(t(src), t(dst), split(ref.proj_q[0], h64), split(ref.proj_k[0], h64), split(ref.proj_v[0], h64), ref.bias_table, t(etype))
    x = ref.norm_in[0](h64 + ref.proj_o[0](a.reshape(-1, 512)))
    a = attention64(t(isrc), t(idst), split(ref.proj_q[1], x), split(ref.proj_k[1], mem64), split(ref.proj_v[1], mem64))
    x = ref.norm_in[1](x + ref.proj_o[1](a.reshape(-1, 512)))
    out64 = ref.norm_inter(x + ref.ffn[0].w_2(torch.relu(ref.ffn[0].w_1(x))))
    out64.backward(gout.double())
    close(out, out64, "block output", 2e-4, 2e-5)
    close(h.grad, h64.grad, "d input", 1e-3, 1e-4)
    close(mem.grad, mem64.grad, "d memory", 1e-3, 1e-4)
    for (name, p), (_, pr) in zip(blk.named_parameters(), ref.named_parameters()):
        close(p.grad, pr.grad, f"d {name}", 1e-3, 1e-4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step_with_all_options_repeats(dtype):
    from bpt_amd.block import BPTBlock
    c = case(500)
    torch.manual_seed(3)
    blk = BPTBlock(512, 8, 1024, drop_h=0.1, drop_a=0.1, score_cap=10.0, distance=True, epilogue=True, bucket_bias=30).to(DEV).to(dtype)
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
    blk.eval()
    assert torch.equal(blk(h, csr, c["etype"].to(DEV), pos), blk(h, csr, c["etype"].to(DEV), pos))


def test_modules_that_are_not_as_they_were_are_called():
    from bpt_amd.block import BPTBlock
    c = case(60)
    csr, h = to_dev(c["csr"]), c["h"].to(DEV)

    def pair():
        torch.manual_seed(3)
        plain = BPTBlock(512, 8, 256, drop_h=0.0, drop_a=0.0).to(DEV)
        other = copy.deepcopy(plain)
        other.epilogue = True
        return plain, other
    plain, other = pair()
    assert (plain(h, csr) - other(h, csr)).abs().max() < 1e-4
    for change in (lambda b: b.proj_o.register_forward_hook(lambda m, i, o: 3 * o), lambda b: b.ffn[0].w_1.register_forward_hook(lambda m, i, o: 3 * o),
                   lambda b: b.ffn.register_forward_hook(lambda m, i, o: 3 * o), lambda b: b.ffn[0].register_forward_hook(lambda m, i, o: 3 * o),
                   lambda b: b.ffn[1].register_forward_hook(lambda m, i, o: 3 * o)):
        plain, other = pair()
        for b in (plain, other):
            change(b)
        assert (plain(h, csr) - other(h, csr)).abs().max() < 1e-4
    plain, other = pair()
    for b in (plain, other):
        b.drop_h.p = b.ffn[1].p = 1.0
    assert torch.equal(plain(h, csr), other(h, csr))
    plain, other = pair()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(plain(h, csr), other(h, csr))
    plain, other = pair()
    assert torch.equal(plain.double()(h.double(), csr), other.double()(h.double(), csr))


def test_projections_with_hooks_are_called():
    from bpt_amd.block import BPTBlock, BPTMemBlock
    c = case(60)
    csr, h = to_dev(c["csr"]), c["h"].to(DEV)
    for kind, args in ((BPTBlock, (h, csr)), (BPTMemBlock, (h, csr, h, csr))):
        for name in ("proj_q", "proj_k", "proj_v"):
            torch.manual_seed(3)
            plain = kind(512, 8, 256, drop_h=0.0, drop_a=0.0).to(DEV)
            other = copy.deepcopy(plain)
            other.epilogue = True
            for b in (plain, other):
                proj = getattr(b, name)
                (proj if kind is BPTBlock else proj[0]).register_forward_hook(lambda m, i, o: 2 * o)
            assert (plain(*args) - other(*args)).abs().max() < 1e-4


def test_a_block_made_without_the_options_and_their_parameters():
    from bpt_amd.block import BPTBlock, BPTMemBlock
    for kind in (BPTBlock, BPTMemBlock):
        assert "bias_table" not in kind(64, 2, 32).state_dict() and kind(64, 2, 32, bucket_bias=7).state_dict()["bias_table"].shape == (7, 2)
        with pytest.raises(ValueError, match="go together"):
            kind(64, 2, 32, rel_pos=True, bucket_bias=7)
    with pytest.raises(ValueError, match="edge types"):
        c = case(20, dim=64)
        BPTBlock(64, 2, 32, bucket_bias=3).to(DEV)(c["h"].to(DEV), to_dev(c["csr"]))
