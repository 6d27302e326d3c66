"""Blocks with bucket_bias under autocast: projections of one type, the table of another."""
import pytest
import torch

from bpt_amd import op
from test_gpu_block_options import case, to_dev

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def block(kind, **opts):
    torch.manual_seed(3)
    blk = kind(512, 8, 256, drop_h=0.0, drop_a=0.0, bucket_bias=12, **opts)
    torch.nn.init.normal_(blk.bias_table)
    return blk.to(DEV)


@pytest.mark.parametrize("opts", [dict(), dict(epilogue=True), dict(score_cap=5.0), dict(fused=False)], ids=str)
def test_the_table_takes_the_projections_type(opts):
    from bpt_amd.block import BPTBlock
    c = case(80)
    csr, h, etype = to_dev(c["csr"]), c["h"].to(DEV), c["etype"].to(DEV)
    blk = block(BPTBlock, **opts)
    out_csr, in_csr, row, indptr_r, col, indptr_c = csr
    with torch.autocast("cuda", dtype=torch.bfloat16):
        q, k, v = (proj(h).view(-1, 8, 64).detach() for proj in (blk.proj_q, blk.proj_k, blk.proj_v))
        assert q.dtype == torch.bfloat16
        got = blk.attention(q, k, v, csr, etype)
    table = blk.bias_table.detach().bfloat16().requires_grad_(True)
    want = op.bpt_attention(row, indptr_r, out_csr[2], out_csr[1], col, indptr_c, in_csr[2], in_csr[1], q, k, v, bias_table=table, buckets=etype,
                            score_cap=opts.get("score_cap"), fused=opts.get("fused")).view(-1, 512)
    assert torch.equal(got, want)
    do = torch.randn_like(want)
    got.backward(do)
    want.backward(do)
    assert blk.bias_table.grad.dtype == torch.float32 and torch.equal(blk.bias_table.grad, table.grad.float()) and table.grad.any()


def test_layers_run_both_ways():
    from bpt_amd.block import BPTBlock, BPTMemBlock
    c = case(80)
    csr, etype = to_dev(c["csr"]), c["etype"].to(DEV)
    for kind in (BPTBlock, BPTMemBlock):
        blk, h = block(kind), c["h"].to(DEV).requires_grad_(True)
        args = (h, csr) if kind is BPTBlock else (h, csr, h, csr)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = blk(*args, etype)
            out.float().square().sum().backward()
        grads = [h.grad] + [p.grad for p in blk.parameters()]
        assert out.isfinite().all() and all(g.isfinite().all() and g.any() for g in grads)
        # as without autocast, but for the type: 2^-8 a rounding, some ten on the way, of outputs that are normalised rows
        assert (out.float() - blk(*args, etype)).abs().max() < 10 * 2.0 ** -8 * 4
