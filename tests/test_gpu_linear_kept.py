"""bpt_linear_forward's kept: the pre-activation in the call's type, whatever the activation and the sizes, and so the way it is formed."""
import pytest
import torch

from test_epilogue_bias_abi import linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(3, 64, 64), (40, 96, 72), (300, 256, 200), (300, 256, 202), (100, 8192, 64), (2000, 256, 1024), (8190, 1100, 1540)], ids=str)
def test_kept_is_what_the_activation_takes(size, dtype):
    rows, inner, outer = size
    gen = torch.Generator().manual_seed(rows)
    x, w, b, r = (torch.randn(shape, generator=gen).to(dtype).to(DEV) for shape in ((rows, inner), (outer, inner), (outer,), (rows, outer)))
    lib, code = linear(), 0 if dtype == torch.float32 else 2
    need = lib.bpt_linear_forward_workspace_bytes(rows, inner, outer, code)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)

    def forward(act, residual, p, kept):
        y = torch.empty(rows, outer, dtype=dtype, device=DEV)
        st = lib.bpt_linear_forward(x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr() if residual else None, y.data_ptr(), None if kept is None else kept.data_ptr(),
                                    ws.data_ptr(), need, rows, inner, outer, act, p, 7, code, torch.cuda.current_stream().cuda_stream)
        assert st == 0
        return y
    a = forward(0, False, 0.0, None)                              # (no activation: the result is the pre-activation)
    for act in (0, 1, 2):
        for residual, p in ((False, 0.0), (True, 0.0), (False, 0.3), (True, 0.3)):
            kept = torch.full_like(a, float("nan"))
            y = forward(act, residual, p, kept)
            assert torch.equal(kept, a), (act, residual, p)
            assert torch.equal(y, forward(act, residual, p, None)), (act, residual, p)
