"""The C ABI of attention with score options and of the block's operators (include/bptscore.h, include/bptblock.h): what is declared is exported, the Python
bindings cover it, and calls that do not fit are refused; and what op.bpt_attention refuses of its score options before anything reaches a GPU."""
import ctypes
import os
import re

import pytest
import torch

from bpt_amd import _build, _lib, op

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def constants():
    text = open(os.path.join(ROOT, "include", "bptattn.h")).read()
    return {n: int(v) for n, v in re.findall(r"(BPT_(?:OK|ERR_\w+))\s*=\s*(-?\d+)", text)}


C = constants()


def declared(header, prefix):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", header)).read(), flags=re.S)
    return sorted(set(re.findall(r"^\s*(?:int|int64_t|const char \*)\s*(" + prefix + r"\w+)\(", text, flags=re.M)))


@pytest.mark.parametrize("header,prefix,so,n", [("bptscore.h", "bpt_score_", _build.SCORE_SO, 4), ("bptblock.h", "bpt_", _build.BLOCK_SO, 5)])
def test_declared_functions_are_exported(header, prefix, so, n):
    names = declared(header, prefix)
    assert len(names) == n
    lib = ctypes.CDLL(so)
    for name in names:
        assert hasattr(lib, name), name


def test_the_bindings_cover_the_declared_functions():
    assert sorted(_lib.SCORE_API) == declared("bptscore.h", "bpt_score_")


def plan(**kw):
    """A plan whose pointers are set and never followed: every call below is refused before a kernel could read them."""
    p = 1 << 20
    d = dict(rowptr=p, idx=p, eid=p, items=p, heavy=None, n_rows=4, n_edges=9, n_items=4, n_heavy=0, n_slots=0, grp_members=p, grp_ptr=p, grp_entries=p,
             grp_pairs=p, grp_chunks=p, n_groups=1, grp_R=16, grp_max_chunk=1, n_grp_entries=9, grp_eids=p, bias_by_pair=0, n_index_nodes=4, max_degree=9)
    return _lib.PlanStruct(**dict(d, **kw))


def forward(pl=None, score=(30.0, None, None, None), q=1 << 20, bias=None, ws=None, ws_bytes=0, scale=0.125, p=0.0, heads=8, d=64, h=8, dtype=0):
    lib, at = _lib.score_lib(), 1 << 20
    pl = plan() if pl is None else pl
    sc = None if score is None else ctypes.byref(_lib.ScoreStruct(*score))
    return lib.bpt_score_forward(ctypes.byref(pl) if pl else None, sc, q, at, at, bias, at, at, ws, ws_bytes, scale, p, 0, heads, d, h, dtype, None)


def test_a_forward_that_does_not_fit_is_refused():
    p = 1 << 20
    assert forward(pl=False) == C["BPT_ERR_NULL"] and forward(score=None) == C["BPT_ERR_NULL"] and forward(q=None) == C["BPT_ERR_NULL"]
    assert forward(pl=plan(n_rows=-1)) == C["BPT_ERR_SIZE"] and forward(pl=plan(idx=None)) == C["BPT_ERR_NULL"]
    assert forward(dtype=7) == C["BPT_ERR_DTYPE"] and forward(dtype=1) == C["BPT_ERR_UNSUPPORTED"]                       # (float64 has no fused kernel)
    assert forward(h=5, heads=5) == C["BPT_ERR_UNSUPPORTED"] and forward(h=4, heads=4, dtype=2) == C["BPT_ERR_UNSUPPORTED"]
    assert forward(heads=0) == C["BPT_ERR_SHAPE"] and forward(d=0) == C["BPT_ERR_SHAPE"]
    for bad in (dict(heads=9), dict(d=3), dict(d=65), dict(heads=6, bias=p), dict(heads=6, d=49, dtype=2)):
        assert forward(**bad) == C["BPT_ERR_UNSUPPORTED"], bad
    for cap in (-1.0, float("inf"), float("nan"), 1e-6, 1e-11, 1e11):
        assert forward(score=(cap, None, None, None)) == C["BPT_ERR_SIZE"], cap
    assert forward(scale=float("nan")) == C["BPT_ERR_SIZE"] and forward(score=(1e9, None, None, None), scale=1e7) == C["BPT_ERR_SIZE"]
    for rate in (-0.1, 1.0, float("nan")):
        assert forward(p=rate) == C["BPT_ERR_SIZE"], rate
    assert forward(score=(0.0, p, None, p)) == C["BPT_ERR_NULL"] and forward(score=(0.0, p, p, None)) == C["BPT_ERR_NULL"]
    assert forward(q=p + 4) == C["BPT_ERR_UNSUPPORTED"] and forward(q=p + 2, heads=6) == C["BPT_ERR_UNSUPPORTED"]
    assert forward(pl=plan(n_groups=0, grp_members=None), p=0.5) == C["BPT_ERR_UNSUPPORTED"]                             # (single rows have no dropout, no bias)
    assert forward(pl=plan(n_groups=0, grp_members=None), heads=6) == C["BPT_ERR_UNSUPPORTED"]
    assert forward(pl=plan(grp_R=8)) == C["BPT_ERR_UNSUPPORTED"] and forward(pl=plan(n_rows=1 << 22, n_items=1 << 22)) == C["BPT_ERR_UNSUPPORTED"]     # (2^33 bytes)
    for bad in (dict(p=0.5), dict(heads=6), dict(bias=p)):
        assert forward(pl=plan(grp_eids=None), **bad) == C["BPT_ERR_PLAN"], bad
    assert forward(pl=plan(bias_by_pair=1), bias=p) == C["BPT_ERR_PLAN"]
    split = plan(heavy=p, n_heavy=1, n_slots=3)
    need = _lib.score_lib().bpt_score_forward_workspace_bytes(ctypes.byref(split), 8)
    assert need == 3 * (8 * 64 + 2 * 8) * 4
    assert forward(pl=split) == C["BPT_ERR_WORKSPACE"] and forward(pl=split, ws=p, ws_bytes=need - 1) == C["BPT_ERR_WORKSPACE"]
    assert forward(pl=plan(n_rows=0, n_edges=0, n_items=0)) == C["BPT_OK"] and forward(pl=plan(n_rows=0, n_items=0)) == C["BPT_ERR_UNSUPPORTED"]


def test_a_backward_that_does_not_fit_is_refused():
    lib, at = _lib.score_lib(), 1 << 20

    def backward(pi=None, po=None, score=(30.0, None, None, None), bias=None, ds=None, dslopes=None, q=at, dk=at, ws=at, ws_bytes=1 << 40, p=0.0, heads=8, d=64, h=8, dtype=0):
        pi, po = plan() if pi is None else pi, plan() if po is None else po
        return lib.bpt_score_backward(ctypes.byref(pi), ctypes.byref(po), ctypes.byref(_lib.ScoreStruct(*score)), q, at, at, bias, at, at, at, at, dk, at, ds, dslopes,
                                      ws, ws_bytes, 0.125, p, 0, heads, d, h, dtype, None)
    assert backward(po=plan(n_edges=8)) == C["BPT_ERR_PLAN"]
    assert backward(po=plan(grp_pairs=None)) == C["BPT_ERR_UNSUPPORTED"] and backward(po=plan(n_groups=0)) == C["BPT_ERR_UNSUPPORTED"]
    assert backward(pi=plan(n_groups=0, grp_members=None)) == C["BPT_ERR_UNSUPPORTED"]
    assert backward(bias=at) == C["BPT_ERR_NULL"] and backward(ds=at) == C["BPT_ERR_NULL"] and backward(dslopes=at) == C["BPT_ERR_NULL"]
    assert backward(p=0.5, dtype=2, po=plan(grp_eids=None)) == C["BPT_ERR_PLAN"]
    assert backward(q=None) == C["BPT_ERR_NULL"] and backward(dk=None) == C["BPT_ERR_NULL"]
    assert backward(dk=at + 8) == C["BPT_ERR_UNSUPPORTED"] and backward(dk=at + 2, heads=6, dtype=2) == C["BPT_ERR_UNSUPPORTED"] and backward(ws=at + 4) == C["BPT_ERR_UNSUPPORTED"]
    for dtype in (0, 2):
        need = lib.bpt_score_backward_workspace_bytes(ctypes.byref(plan()), ctypes.byref(plan()), 8, dtype, 0)
        assert need > 0 and backward(dtype=dtype, ws_bytes=need - 1) == C["BPT_ERR_WORKSPACE"] and backward(dtype=dtype, ws=None) == C["BPT_ERR_WORKSPACE"]
    assert lib.bpt_score_backward_workspace_bytes(None, None, 8, 0, 0) == -1 and lib.bpt_score_backward_workspace_bytes(ctypes.byref(plan()), ctypes.byref(plan()), 8, 1, 0) == -1


def test_what_the_operator_refuses():
    e = torch.zeros(3, dtype=torch.int64)
    ptr = torch.tensor([0, 1, 2, 3])
    graph = (e, ptr, e, e, e, ptr, e, e)
    q = torch.randn(3, 8, 64)
    go = lambda **kw: op.bpt_attention(*graph, q, q, q, **kw)
    for cap in (0.0, -2.0, float("inf"), float("nan"), 1e-9, 1e-11, 1e11):
        with pytest.raises(ValueError, match="score_cap"):
            go(score_cap=cap)
    with pytest.raises(ValueError, match="go together"):
        go(slopes=torch.ones(8))
    with pytest.raises(ValueError, match="go together"):
        go(pos=torch.ones(3))
    with pytest.raises(ValueError, match="pair"):
        go(slopes=torch.ones(8), pos=(torch.ones(3),) * 3)
    with pytest.raises(ValueError, match="rel_table and etype"):
        go(score_cap=3.0, rel_table=torch.ones(2, 64))
    for opts in (dict(score_cap=3.0), dict(slopes=torch.ones(8), pos=torch.ones(3))):
        with pytest.raises(RuntimeError, match="CUDA"):
            go(**opts)
