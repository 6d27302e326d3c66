"""Blocks with bucket_bias whose table has been learned, against the formula.  Tolerances as in the tests of the other options."""
import copy

import pytest
import torch

from test_gpu_block_epilogue import attention64
from test_gpu_block_options import case, close, to_dev

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("epilogue", [False, True])
@pytest.mark.parametrize("dims", [(512, 8, 256), (300, 6, 130), (96, 3, 64), (160, 2, 64)], ids=str)
def test_block_with_a_learned_table(dims, epilogue):
    from bpt_amd.block import BPTBlock
    dim, heads, ff = dims
    c = case(dim=dim)
    torch.manual_seed(7)
    blk = BPTBlock(dim, heads, ff, drop_h=0.0, drop_a=0.0, epilogue=epilogue, bucket_bias=12)
    blk.reset_parameters()
    torch.nn.init.normal_(blk.bias_table)
    ref = copy.deepcopy(blk).double()
    blk = blk.to(DEV)
    h = c["h"].to(DEV).requires_grad_(True)
    out = blk(h, to_dev(c["csr"]), c["etype"].to(DEV))
    out.backward(c["gout"].to(DEV))
    h64 = c["h"].double().requires_grad_(True)
    split = lambda proj: proj(h64).view(-1, heads, dim // heads)
    a = attention64(c["src"], c["dst"], split(ref.proj_q), split(ref.proj_k), split(ref.proj_v), ref.bias_table, c["etype"])
    x = ref.norm_in(h64 + ref.proj_o(a.reshape(-1, dim)))
    out64 = ref.norm_inter(x + ref.ffn[0].w_2(torch.relu(ref.ffn[0].w_1(x))))
    out64.backward(c["gout"].double())
    close(out, out64, "block output", 2e-4, 2e-5)
    close(h.grad, h64.grad, "d input", 1e-3, 1e-4)
    for (name, p), (_, pr) in zip(blk.named_parameters(), ref.named_parameters()):
        close(p.grad, pr.grad, f"d {name}", 1e-3, 1e-4)
