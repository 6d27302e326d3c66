"""The C ABI of products with an epilogue, dropout and biases by buckets (include/bptlinear.h, include/bptbias.h): what is declared is exported and calls that do not
fit are refused before anything is launched; and what op.linear_act, op.dropout, op.bucket_bias and op.bpt_attention with a bias refuse without a GPU."""
import ctypes

import pytest
import torch

from bpt_amd import _build, _lib, op
from test_score_abi import C, declared, plan

AT = 1 << 20                                                      # (never read: every call is refused, or has nothing to do)
f32, i32, i64, u64, vp, f64 = ctypes.c_float, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_double
OK, NULL, SIZE, DTYPE, UNSUPPORTED, WORKSPACE, PLAN = (C["BPT_" + n] for n in ("OK", "ERR_NULL", "ERR_SIZE", "ERR_DTYPE", "ERR_UNSUPPORTED", "ERR_WORKSPACE", "ERR_PLAN"))


@pytest.mark.parametrize("header,so,n", [("bptlinear.h", _build.LINEAR_SO, 9), ("bptbias.h", _build.BIAS_SO, 8)])
def test_declared_functions_are_exported(header, so, n):
    names = declared(header, "bpt_")
    assert len(names) == n
    lib = ctypes.CDLL(so)
    for name in names:
        assert hasattr(lib, name), name


def test_the_bindings_cover_the_declared_functions():
    assert sorted(_lib.BIAS_API) == declared("bptbias.h", "bpt_")


def linear():
    lib = ctypes.CDLL(_build.LINEAR_SO)
    lib.bpt_linear_forward.argtypes = [vp] * 7 + [i64] * 4 + [i32, f64, u64, i32, vp]
    lib.bpt_linear_grad.argtypes = [vp, vp, i32] + [vp] * 3 + [i64] * 3 + [i32, f64, u64, i32, vp]
    for name in ("forward", "input_grad", "weight_grad"):
        size = getattr(lib, f"bpt_linear_{name}_workspace_bytes")
        size.argtypes, size.restype = [i64] * 3 + [i32], i64
    lib.bpt_linear_grad_workspace_bytes.argtypes, lib.bpt_linear_grad_workspace_bytes.restype = [i64, i64, i32], i64
    for call in (lib.bpt_linear_input_grad, lib.bpt_linear_weight_grad):
        call.argtypes = [vp] * 4 + [i64] * 4 + [f64, i32, vp]
    lib.bpt_dropout.argtypes = [vp] * 3 + [i64, f64, u64, i32, vp]
    return lib


def test_linear_checks_its_arguments():
    lib = linear()

    def forward(x=AT, w=AT, y=AT, ws=None, ws_bytes=0, rows=4, inner=8, outer=8, act=0, p=0.0, dtype=0):
        return lib.bpt_linear_forward(x, w, None, None, y, None, ws, ws_bytes, rows, inner, outer, act, p, 0, dtype, None)
    for bad in (dict(x=None), dict(w=None), dict(y=None)):
        assert forward(**bad) == NULL, bad
    for bad in (dict(rows=-1), dict(inner=0), dict(outer=-2), dict(rows=(1 << 28) + 1), dict(rows=1 << 28, outer=1 << 20), dict(p=1.0), dict(p=-0.1), dict(p=float("nan"))):
        assert forward(**bad) == SIZE, bad
    assert forward(dtype=1) == DTYPE and forward(dtype=9) == DTYPE and forward(act=3) == UNSUPPORTED and forward(act=-1) == UNSUPPORTED
    assert forward(x=None, rows=0) == OK and forward(y=None, outer=0) == OK
    size = lib.bpt_linear_forward_workspace_bytes
    assert size(-1, 8, 8, 0) == -1 and size(8, 8, 8, 1) == -1 and size(4, 1 << 20, 8, 0) == 0
    shape = dict(rows=100, inner=1 << 16, outer=64)
    need = size(100, 1 << 16, 64, 0)
    assert need > 0                                               # (a long reduction of one tile is shared)
    for bad in (dict(), dict(ws=AT, ws_bytes=need - 1), dict(ws=AT + 4, ws_bytes=need)):
        assert forward(**shape, **bad) == WORKSPACE, bad

    def grad(dy=AT, kept=AT, g=AT, db=None, ws=None, ws_bytes=0, rows=4, outer=8, act=1, p=0.0, dtype=0):
        return lib.bpt_linear_grad(dy, kept, 0, g, db, ws, ws_bytes, rows, outer, act, p, 0, dtype, None)
    assert grad(dy=None) == NULL and grad(kept=None) == NULL and grad(rows=-1) == SIZE and grad(p=1.0) == SIZE and grad(dtype=1) == DTYPE and grad(act=7) == UNSUPPORTED
    need = lib.bpt_linear_grad_workspace_bytes(4, 8, 0)
    assert need > 0 and grad(db=AT, ws=AT, ws_bytes=need - 1) == WORKSPACE and grad(db=AT) == WORKSPACE
    for call in (lib.bpt_linear_input_grad, lib.bpt_linear_weight_grad):
        go = lambda a=AT, b=AT, c=AT, rows=4, inner=8, outer=8, dtype=0: call(a, b, c, None, 0, rows, inner, outer, 1.0, dtype, None)
        assert go(a=None) == NULL and go(b=None) == NULL and go(c=None) == NULL and go(rows=-1) == SIZE and go(inner=-1) == SIZE and go(dtype=1) == DTYPE
    drop = lambda x=AT, y=AT, n=8, p=0.5, dtype=0: lib.bpt_dropout(x, None, y, n, p, 0, dtype, None)
    assert drop(x=None) == NULL and drop(y=None) == NULL and drop(n=-1) == SIZE and drop(p=1.0) == SIZE and drop(dtype=1) == DTYPE and drop(x=None, n=0) == OK


def ref(p):
    return None if p is None else ctypes.byref(p)


def test_biases_check_their_arguments():
    lib = _lib.bias_lib()
    fwd = lambda table=AT, buckets=AT, bias=AT, n=4, m=3, h=8, spare=0, dtype=0, out=0: lib.bpt_bucket_bias_forward(table, buckets, bias, n, m, h, 1.0, spare, dtype, out, None)
    assert fwd(table=None) == NULL and fwd(buckets=None) == NULL and fwd(bias=None) == NULL and fwd(dtype=9) == DTYPE and fwd(dtype=0, out=2) == DTYPE
    assert fwd(n=-1) == SIZE and fwd(m=0) == SIZE and fwd(h=0) == SIZE and fwd(spare=2) == SIZE and fwd(table=None, n=0) == OK
    bwd = lambda ds=AT, dt=AT, ws=AT, nws=1 << 40, n=4, dtype=0: lib.bpt_bucket_bias_backward(ds, AT, dt, ws, nws, n, 3, 8, 1.0, dtype, dtype, None)
    assert bwd(ds=None) == NULL and bwd(dt=None) == NULL and bwd(ws=None) == WORKSPACE and bwd(nws=0) == WORKSPACE and bwd(ws=AT + 4) == WORKSPACE and bwd(dtype=9) == DTYPE

    def prepare(pi=plan(), po=None, table=AT, buckets=AT, m=3, heads=8, h=8, scale=0.1, dtype=0, to=AT):
        return lib.bpt_bucket_prepare(ref(pi), ref(po), table, buckets, m, heads, h, scale, dtype, to, None)
    assert prepare(pi=None) == NULL and prepare(table=None) == NULL and prepare(buckets=None) == NULL and prepare(to=None) == NULL and prepare(to=AT + 8) == UNSUPPORTED
    assert prepare(dtype=1) == DTYPE
    for bad in (dict(m=0), dict(m=256), dict(heads=0), dict(heads=9), dict(h=17, heads=17), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert prepare(**bad) == SIZE, bad
    for bad in (dict(pi=plan(grp_eids=None)), dict(po=plan(grp_eids=None)), dict(pi=plan(grp_R=8)), dict(po=plan(n_edges=8)), dict(po=plan(n_groups=0)),
                dict(pi=plan(n_groups=0), po=plan())):
        assert prepare(**bad) == PLAN, bad
    size = lib.bpt_bucket_prepare_bytes
    assert size(None, None, 8) == -1 and size(ref(plan()), None, 0) == -1 and size(ref(plan()), None, 17) == -1
    assert size(ref(plan()), None, 8) == 8 * 1024 + 9 * 16 and size(ref(plan()), ref(plan()), 8) == 8 * 1024 + 2 * 9 * 16 + 16

    def attend(pl=plan(), score=(0.0, None, None, None), prepared=AT, q=AT, lse=AT, ws=None, nws=0, p=0.0, h=8, dtype=0):
        return lib.bpt_bucket_attention_forward(ref(pl), None if score is None else ctypes.byref(_lib.ScoreStruct(*score)), prepared, q, AT, AT, AT, lse, ws, nws, 0.125, p,
                                                0, h, dtype, None)
    assert attend(pl=None) == NULL and attend(score=None) == NULL and attend(prepared=None) == NULL and attend(q=None) == NULL and attend(lse=None) == NULL
    assert attend(h=5) == UNSUPPORTED and attend(h=4, dtype=2) == UNSUPPORTED and attend(dtype=1) == UNSUPPORTED and attend(dtype=7) == DTYPE
    assert attend(p=1.0) == SIZE and attend(score=(-1.0, None, None, None)) == SIZE and attend(q=AT + 4) == UNSUPPORTED and attend(pl=plan(grp_eids=None)) == PLAN
    assert attend(pl=plan(heavy=AT, n_heavy=1, n_slots=3)) == WORKSPACE and attend(pl=plan(n_rows=0, n_edges=0, n_items=0)) == OK

    def back(pi=plan(), po=plan(), score=(0.0, None, None, None), prepared=AT, dk=AT, dtable=AT, dslopes=None, ws=AT, nws=1 << 40, m=3, heads=8, dtype=0):
        return lib.bpt_bucket_attention_backward(ref(pi), ref(po), ctypes.byref(_lib.ScoreStruct(*score)), prepared, AT, AT, AT, AT, AT, AT, AT, dk, AT, dtable, dslopes, ws,
                                                 nws, m, heads, 0.125, 0.0, 0, 8, dtype, None)
    assert back(pi=None) == NULL and back(po=None) == NULL and back(prepared=None) == NULL and back(dk=None) == NULL and back(dslopes=AT) == NULL
    assert back(m=0) == SIZE and back(m=256) == SIZE and back(heads=9) == SIZE and back(dk=AT + 8) == UNSUPPORTED and back(po=plan(grp_pairs=None)) == UNSUPPORTED
    for bad in (dict(po=plan(n_edges=8)), dict(pi=plan(grp_eids=None)), dict(po=plan(grp_eids=None))):
        assert back(**bad) == PLAN, bad
    assert back(pi=plan(n_groups=0)) == UNSUPPORTED and back(ws=None) == WORKSPACE
    size = lib.bpt_bucket_attention_backward_workspace_bytes
    for dtype in (0, 2):
        need = size(ref(plan()), ref(plan()), 3, 8, 8, dtype)
        assert need > 0 and back(dtype=dtype, nws=need - 1) == WORKSPACE
    assert size(None, None, 3, 8, 8, 0) == -1 and size(ref(plan()), ref(plan()), 256, 8, 8, 0) == -1 and size(ref(plan()), ref(plan()), 3, 9, 8, 0) == -1


def test_what_the_operators_refuse():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    for go in (lambda: op.linear_act(x, w), lambda: op.dropout(x, 0.1), lambda: op.bucket_bias(torch.randn(3, 8), torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            go()
    with pytest.raises(ValueError, match="activation"):
        op.linear_act(x, w, activation="tanh")
    for call in (lambda t: op.linear_act(t, w), lambda t: op.dropout(t, 0.5)):
        with pytest.raises(RuntimeError, match="transforms"):
            torch.func.vmap(call)(torch.randn(3, 4, 8))
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.vmap(lambda t: op.bucket_bias(t, torch.zeros(4, dtype=torch.int64)))(torch.randn(2, 3, 8))
    e, at = torch.zeros(3, dtype=torch.int64), torch.tensor([0, 1, 2, 3])
    q = torch.randn(3, 8, 64)
    go = lambda **kw: op.bpt_attention(e, at, e, e, e, at, e, e, q, q, q, **kw)
    for match, kw in [("go together", dict(bias_table=torch.ones(2, 8))), ("go together", dict(buckets=e)), ("bias_table must be", dict(bias_table=torch.ones(2, 7), buckets=e)),
                      ("one element for every edge", dict(bias_table=torch.ones(2, 8), buckets=e[:2])), ("score_cap", dict(bias_table=torch.ones(2, 8), buckets=e, score_cap=-1.0))]:
        with pytest.raises(ValueError, match=match):
            go(**kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        go(bias_table=torch.ones(2, 8), buckets=e)
