"""The slopes' gradient of bfloat16 attention with relative positions where a few rows are split, as the nodes near the root of a binary partition are.

Nothing that it is summed from is rounded to bfloat16, so it meets float32's bound of the same values (test_gpu_score_attention).  The values are such that a
delta formed from o as stored is far outside: v is 1 or, three times in ten, 1 + 2^-7, so o is 1 + 0.3 * 2^-7 and is stored as 1 in every column, and do is positive.  Scores are small
and the slopes times the distances below one: p is even, which leaves float32's bound near (edges of a row) * 2^-24 of a row's sum."""
import pytest
import torch

from test_gpu_score_attention import close, graph_args, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,d", [(8, 64), (16, 64), (6, 50)])
@pytest.mark.parametrize("long_rows", [1, 10, 100])
def test_few_split_rows(long_rows, heads, d):
    """All edges of 1000 nodes lead to a few of them."""
    from bpt_amd import graphop
    c = make(("random", 1000, 1500 * long_rows), heads, d, "bf16", 15.0, True, rel=True, q_scale=0.1)
    c["dst"] = c["dst"] % long_rows * 7
    gen = torch.Generator().manual_seed(4)
    draw = lambda name: torch.rand(c[name].shape, generator=gen)
    c["v"] = (1 + (draw("v") < 0.3).float() * 2.0 ** -7).bfloat16()
    c["do"] = ((1 + draw("do")) / 16).bfloat16()
    c["slopes"] = (1 + torch.rand(heads, generator=gen)) / (8 * c["q"].size(0))
    args = graph_args(c["src"].numpy(), c["dst"].numpy(), c["q"].size(0), c["k"].size(0))
    got = run(c, args, True)
    like = torch.empty((c["q"].size(0), graphop.score_padded_shape(c["q"])[0], 64), dtype=torch.bfloat16, device=args[0].device)
    plan = graphop._score_plan_in(args, like, like)
    assert 0 < 2 * plan.struct.n_heavy < plan.struct.n_rows       # some rows are split, most are not
    wide = {n: t.float() if torch.is_tensor(t) and t.dtype == torch.bfloat16 else t for n, t in c.items()}
    want = reference(wide)["dslopes"]
    close(got["dslopes"], want, "dslopes", torch.float32)
