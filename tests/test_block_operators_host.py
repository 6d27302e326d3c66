"""What op.add_layer_norm, op.relu_linear8 and graphop.relu8_* refuse without a GPU, and the C ABI's own checks."""
import ctypes

import pytest
import torch

from bpt_amd import _build, graphop, op


def test_host_tensors_are_refused():
    x = torch.randn(4, 64)
    for call in (lambda: op.add_layer_norm(x), lambda: op.relu_linear8(x, torch.randn(8, 64)), lambda: graphop.relu8_forward(x),
                 lambda: graphop.relu8_backward(x, torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, dtype=torch.int8))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_transforms_are_refused():
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.vmap(lambda x: op.add_layer_norm(x))(torch.randn(3, 4, 8))


def test_c_abi_checks_its_arguments():
    lib = ctypes.CDLL(_build.BLOCK_SO)
    i64, vp, f, d, i = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_double, ctypes.c_int
    fwd, bwd, size = lib.bpt_add_norm_forward, lib.bpt_add_norm_backward, lib.bpt_add_norm_workspace_bytes
    fwd.argtypes, bwd.argtypes = [vp] * 6 + [i64, i64, d, i, vp], [vp] * 9 + [i64, i64, i64, i, vp]
    size.argtypes, size.restype = [i64, i64, i], i64
    NULL, SIZE, DTYPE, WORKSPACE = -1, -2, -3, -5
    p = 1 << 20                                                   # (never read: every call is refused, or has nothing to do)
    assert fwd(None, None, None, None, None, None, 4, 64, 1e-5, 0, None) == NULL
    assert fwd(p, None, None, None, p, None, -1, 64, 1e-5, 0, None) == SIZE
    assert fwd(p, None, None, None, p, None, 4, 0, 1e-5, 0, None) == SIZE
    assert fwd(p, None, None, None, p, None, 4, 64, 1e-5, 7, None) == DTYPE
    assert fwd(None, None, None, None, None, None, 0, 64, 1e-5, 0, None) == 0
    assert bwd(p, None, None, p, p, p, p, p, None, 0, 4, 64, 0, None) == WORKSPACE
    assert bwd(p, None, None, p, p, p, p, p, p, size(4, 64, 0) - 1, 4, 64, 0, None) == WORKSPACE
    assert bwd(p, None, None, None, p, p, None, None, None, 0, 4, 64, 0, None) == NULL
    assert bwd(p, None, None, p, p, None, None, None, None, 0, 4, 64, 0, None) == 0
    assert size(-1, 64, 0) < 0 and size(4, 64, 9) < 0 and size(1 << 20, 512, 0) == 512 * 2 * 512 * 4
    rf, rb = lib.bpt_relu8_forward, lib.bpt_relu8_backward
    rf.argtypes, rb.argtypes = [vp] * 4 + [i64, f, ctypes.c_uint64, i, vp], [vp] * 5 + [i64, f, i, vp]
    assert rf(p, p, p, p, 64, 0.0, 0, 1, None) == DTYPE
    assert rf(p, p, p, p, -1, 0.0, 0, 0, None) == SIZE and rf(p, p, p, p, 64, 1.0, 0, 0, None) == SIZE
    assert rf(p, p, p, p, (1 << 32) + 1, 0.5, 0, 0, None) == SIZE
    assert rf(None, p, p, p, 64, 0.0, 0, 0, None) == NULL and rf(None, None, None, None, 0, 0.0, 0, 0, None) == 0
    assert rb(None, p, p, p, p, 64, 0.0, 0, None) == NULL and rb(p, p, p, None, None, 64, 0.0, 0, None) == 0
