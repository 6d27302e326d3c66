"""The transformer block of the reference (modules/attention.py:22-81) on the HIP attention kernels.

Same sub-modules, parameter names and initialisation as the reference's `BPTBlock`, so its
`state_dict` loads here unchanged: `norm_in`, `norm_inter`, `proj_q/k/v/o` (bias-free), `embed_ak`
(when `rel_pos`), `ffn.0.w_1`, `ffn.0.w_2`.  The reference keeps node features and edge types in a
DGL graph object (`g.ndata['h']`, `g.edata['etype']`) and writes the result back into it; here
`forward(h, csr, etype)` takes and returns plain tensors, `csr` being the 6-tuple that
`graph/base.py:71-86` (`bpt_amd.graphbuilder.get_csrs`) produces.

Attention core: the fused kernels (`op.bpt_attention`: rel_pos term and attention dropout included), or with
`fused=False` the four operators composed exactly as attention.py:66-77 does.
Residual and LayerNorm: one kernel each way (`op.add_layer_norm`) on GPU tensors of one type and rows of up to 16 KiB, the torch module
otherwise and with `fused=False`.  Projections and the feed-forward are torch modules (rocBLAS GEMMs).

Options the reference does not have, off by default (then nothing of them is a parameter, and the results are the reference's):
  score_cap   attention scores become cap tanh(score / cap)
  distance    scores fall by slopes[head] times the distance of the nodes' positions, which `forward` is given as `pos` (float32); `slopes`
              (heads,) is a parameter that starts at 2^(-8 i / heads), i = 1 .. heads
  keep8       the feed-forward keeps its activations in 8 bits for the backward (`op.relu_linear8`): one byte each in place of relu's
              result, dropout's and its mask
"""
import math

import torch
import torch.nn as nn

from .op import (add_layer_norm, bpt_attention, edge_type_embedding, masked_mm, node_mul_edge, plain_call, relu_linear8, sparse_softmax,
                 vec_spmm)

__all__ = ["PositionwiseFeedForward", "BPTBlock", "BPTMemBlock"]


def _as_it_is(module, kind):
    """Whether a call of module is the forward of kind, a class of torch.nn, and nothing else."""
    return (type(module) is kind and "forward" not in module.__dict__
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks)
            and not nn.modules.module._has_any_global_hook())


def _add_norm(norm, x, residual, fused):
    """norm(x + residual) (attention.py:79, :81), by add_layer_norm where that computes the same and is the faster way: a LayerNorm over the last axis as it is,
    GPU tensors of one type, nothing that casts, traces or transforms, rows that a workgroup's registers hold (16 KiB).  Longer rows are walked three times:
    forward | training, us, add_layer_norm / torch, 16383 rows of 4096 columns float32 145 / 263 | 352 / 736, of 4104 301 / 275 | 767 / 782; of 8192 columns
    bfloat16 152 / 305 | 378 / 898, of 8200 757 / 317 | 1952 / 955; in float64, where torch's is slower, of 2048 columns 146 / 381 | 370 / 843, of 4104 515 / 730 | 1345 / 1556."""
    if (fused and _as_it_is(norm, nn.LayerNorm) and len(norm.normalized_shape) == 1 and x.is_cuda and x.is_contiguous()
            and x.dtype in (torch.float32, torch.float64, torch.bfloat16) and x.dim() > 0 and x.size(-1) == norm.normalized_shape[0]
            and (x.dtype == torch.float64 or x.size(-1) * x.element_size() <= 16384) and x.shape == residual.shape and not torch.is_autocast_enabled()
            and all(t is None or (t.dtype == x.dtype and t.device == x.device and t.is_contiguous()) for t in (residual, norm.weight, norm.bias))
            and plain_call(x, residual, norm.weight, norm.bias)):
        return add_layer_norm(x, residual, norm.weight, norm.bias, norm.eps)
    return norm(x + residual)


def _distance_slopes(h):
    return nn.Parameter(2.0 ** (-8.0 * torch.arange(1, h + 1, dtype=torch.float32) / h))


def _score_options(block, pos):
    """bpt_attention's score options of a block."""
    opts = {}
    if block.score_cap is not None:
        opts["score_cap"] = block.score_cap
    if block.distance:
        if pos is None:
            raise ValueError("distance=True needs the positions of the nodes (pos)")
        opts.update(slopes=block.slopes.float(), pos=pos)
    return opts


class PositionwiseFeedForward(nn.Module):
    """FFN(x) = max(0, x W_1 + b_1) W_2 + b_2   (modules/attention.py:8-19).  keep8: the activations are kept in 8 bits for the backward, where they are
    float32 or bfloat16 GPU tensors and nothing traces or transforms the call."""

    keep8 = False           # (also of a module that was pickled without the option)

    def __init__(self, dim_model, dim_ff, dropout=0.1, keep8=False):
        super().__init__()
        self.keep8 = keep8
        self.w_1 = nn.Linear(dim_model, dim_ff)
        self.w_2 = nn.Linear(dim_ff, dim_model)
        self.dropout = nn.Dropout(dropout)

    def forward(self, x):
        a = self.w_1(x)
        # (modules that someone has replaced, hooked or told to drop everything are called)
        if self.keep8 and a.is_cuda and _as_it_is(self.w_2, nn.Linear) and _as_it_is(self.dropout, nn.Dropout) and not self.dropout.p >= 1.0:
            w, b, cast = self.w_2.weight, self.w_2.bias, torch.is_autocast_enabled()
            if cast:
                w, b = w.to(a.dtype), None if b is None else b.to(a.dtype)
            if (a.dtype in (torch.float32, torch.bfloat16) and not (cast and a.dtype != torch.get_autocast_dtype("cuda")) and a.dim() > 0 and a.size(-1) > 0
                    and all(t is None or (t.dtype == a.dtype and t.device == a.device and t.is_contiguous()) for t in (w, b)) and plain_call(a, w, b)):
                return relu_linear8(a.contiguous(), w, b, self.dropout.p if self.training else 0.0)
        return self.w_2(self.dropout(torch.relu(a)))


class BPTBlock(nn.Module):
    MAX_ETYPE = 1000        # modules/attention.py:23
    score_cap, distance = None, False

    def __init__(self, dim_model, h, dim_ff, rel_pos=False, drop_h=0.1, drop_a=0.1, fused=True, score_cap=None, distance=False, keep8=False):
        super().__init__()
        self.fused = fused          # False: the four operators composed exactly as attention.py:66-77 does
        self.score_cap, self.distance = score_cap, distance
        self.dim_model, self.h, self.dim_ff = dim_model, h, dim_ff
        self.d_k = dim_model // h
        self.rel_pos = rel_pos
        self.drop_h = nn.Dropout(drop_h)
        self.drop_att = nn.Dropout(drop_a)
        self.norm_in = nn.LayerNorm(dim_model)
        self.norm_inter = nn.LayerNorm(dim_model)
        self.proj_q = nn.Linear(dim_model, self.d_k * h, bias=False)
        self.proj_k = nn.Linear(dim_model, self.d_k * h, bias=False)
        self.proj_v = nn.Linear(dim_model, self.d_k * h, bias=False)
        self.proj_o = nn.Linear(self.d_k * h, dim_model, bias=False)
        if rel_pos:
            self.embed_ak = nn.Embedding(self.MAX_ETYPE, self.d_k)
        if distance:
            self.slopes = _distance_slopes(h)
        self.ffn = nn.Sequential(PositionwiseFeedForward(dim_model, dim_ff, dropout=drop_h, keep8=keep8), nn.Dropout(drop_h))

    def reset_parameters(self):
        # modules/attention.py:49-52
        for p in self.parameters():
            if p.dim() > 1:
                nn.init.xavier_uniform_(p)

    def attention(self, q, k, v, csr, etype=None, pos=None):
        """attention.py:66-77: (n, h, d_k) q, k, v -> (n, h * d_k)."""
        out_csr, in_csr, ROW, INDPTR_R, COL, INDPTR_C = csr
        graph = (ROW, INDPTR_R, out_csr[2], out_csr[1], COL, INDPTR_C, in_csr[2], in_csr[1])
        att_dropout = self.drop_att.p if self.training else 0.0
        if self.rel_pos and etype is None:
            raise ValueError("rel_pos=True needs the edge types (etype)")
        opts = _score_options(self, pos)
        if self.fused or opts:
            rel = dict(rel_table=self.embed_ak.weight, etype=etype) if self.rel_pos else {}
            return bpt_attention(*graph, q, k, v, fused=None if self.fused else False, dropout_p=att_dropout, **rel, **opts).view(-1, self.d_k * self.h)
        e = masked_mm(*graph, k, q)
        if self.rel_pos:
            e = e + node_mul_edge(COL, INDPTR_C, in_csr[2], q, edge_type_embedding(self.embed_ak.weight, etype))
        e = self.drop_att(sparse_softmax(COL, INDPTR_C, in_csr[2], e / math.sqrt(self.d_k)))
        return vec_spmm(COL, INDPTR_C, in_csr[2], in_csr[1], ROW, INDPTR_R, out_csr[2], out_csr[1], e, v).view(
            -1, self.d_k * self.h)

    def forward(self, h, csr, etype=None, pos=None):
        # three GEMMs: one strided-batched GEMM over the stacked weights (its (3, n, h * d_k) result holds q, k, v as the
        # contiguous tensors the kernels need) measured slower, 3.38 against 3.17 ms per layer fwd+bwd at n = 16 383 in float32
        q = self.proj_q(h).view(-1, self.h, self.d_k)
        k = self.proj_k(h).view(-1, self.h, self.d_k)
        v = self.proj_v(h).view(-1, self.h, self.d_k)
        a = self.attention(q, k, v, csr, etype, pos) if pos is not None else self.attention(q, k, v, csr, etype)
        h = _add_norm(self.norm_in, h, self.drop_h(self.proj_o(a)), self.fused)
        return _add_norm(self.norm_inter, h, self.ffn(h), self.fused)


def _graph_args(csr):
    out_csr, in_csr, ROW, INDPTR_R, COL, INDPTR_C = csr
    return (ROW, INDPTR_R, out_csr[2], out_csr[1], COL, INDPTR_C, in_csr[2], in_csr[1])


class BPTMemBlock(nn.Module):
    """The decoder-side block of the reference (modules/attention.py:84-172): self-attention over the block's own
    graph, then attention to a memory (encoder states) over an inter graph, then the feed-forward.  Same sub-modules,
    parameter names and initialisation as the reference's `BPTMemBlock` (`proj_q.0` ... `proj_o.1`, `norm_in.0/1`,
    `norm_inter`, `embed_ak`, `ffn.0.w_1/w_2`), so its `state_dict` loads unchanged.

    forward(h, csr, mem, csr_inter, etype=None, pos=None): h (n, dim_model) states of this block's nodes, mem (n_mem, dim_model)
    the memory, csr / csr_inter the 6-tuples of get_csrs; returns the new (n, dim_model) states.  csr_inter may be

      * the reference's square form (graph/mt.py:340-344): both CSRs over max(n, n_mem) nodes.  Queries are then
        padded with zero rows up to the in-CSR's row count as attention.py:148-149 does, and cut back afterwards; or
      * the bipartite form of graphbuilder.get_csrs_bipartite: out-CSR over the n_mem memory nodes, in-CSR over the n
        query nodes; nothing is padded (and n > n_mem, which the reference cannot run, works too).

    Both attention cores run the fused kernels (`op.bpt_attention`) where they cover the shape; `fused=False` composes
    the four operators exactly as the reference does.  score_cap caps the scores of both, distance (with forward's pos, the positions of this
    block's nodes) lowers those of the self-attention; keep8 as in BPTBlock."""
    MAX_ETYPE = 1000        # modules/attention.py:85
    score_cap, distance = None, False

    def __init__(self, dim_model, h, dim_ff, rel_pos=False, drop_h=0.1, drop_a=0.1, fused=True, score_cap=None, distance=False, keep8=False):
        super().__init__()
        self.fused = fused
        self.score_cap, self.distance = score_cap, distance
        self.dim_model, self.h, self.dim_ff = dim_model, h, dim_ff
        self.d_k = dim_model // h
        self.rel_pos = rel_pos
        self.drop_h = nn.ModuleList([nn.Dropout(drop_h) for _ in range(2)])
        self.drop_att = nn.ModuleList([nn.Dropout(drop_a) for _ in range(2)])
        self.norm_in = nn.ModuleList([nn.LayerNorm(dim_model) for _ in range(2)])
        self.norm_inter = nn.LayerNorm(dim_model)
        lin = lambda i, o: nn.ModuleList([nn.Linear(i, o, bias=False) for _ in range(2)])
        self.proj_q, self.proj_k, self.proj_v = (lin(dim_model, self.d_k * h) for _ in range(3))
        self.proj_o = lin(self.d_k * h, dim_model)
        if rel_pos:
            self.embed_ak = nn.Embedding(self.MAX_ETYPE, self.d_k)
        if distance:
            self.slopes = _distance_slopes(h)
        self.ffn = nn.Sequential(PositionwiseFeedForward(dim_model, dim_ff, dropout=drop_h, keep8=keep8), nn.Dropout(drop_h))

    def reset_parameters(self):
        # modules/attention.py:112-115
        for p in self.parameters():
            if p.dim() > 1:
                nn.init.xavier_uniform_(p)

    def _attend(self, which, q, k, v, csr, etype=None, pos=None):
        """attention.py:130-141 (which = 0, with rel_pos) and :156-163 (which = 1): (n_q, h, d_k) -> (n_q, h * d_k)."""
        graph = _graph_args(csr)
        drop = self.drop_att[which]
        p = drop.p if self.training else 0.0
        rel = self.rel_pos and which == 0
        if rel and etype is None:
            raise ValueError("rel_pos=True needs the edge types (etype)")
        opts = _score_options(self, pos) if which == 0 else {} if self.score_cap is None else dict(score_cap=self.score_cap)
        if self.fused or opts:
            extra = dict(rel_table=self.embed_ak.weight, etype=etype) if rel else {}
            return bpt_attention(*graph, q, k, v, fused=None if self.fused else False, dropout_p=p, **extra, **opts).view(-1, self.d_k * self.h)
        COL, INDPTR_C, in_eid, in_idx = graph[4:]
        e = masked_mm(*graph, k, q)
        if rel:
            e = e + node_mul_edge(COL, INDPTR_C, in_eid, q, edge_type_embedding(self.embed_ak.weight, etype))
        e = drop(sparse_softmax(COL, INDPTR_C, in_eid, e / math.sqrt(self.d_k)))
        return vec_spmm(COL, INDPTR_C, in_eid, in_idx, *graph[:4], e, v,
                        n_rows=None if q.size(0) == v.size(0) else q.size(0)).view(-1, self.d_k * self.h)

    def forward(self, h, csr, mem, csr_inter, etype=None, pos=None):
        heads = lambda proj, x: proj(x).view(-1, self.h, self.d_k)
        # Part I: self-attention (attention.py:118-142)
        a = self._attend(0, heads(self.proj_q[0], h), heads(self.proj_k[0], h), heads(self.proj_v[0], h), csr, etype, pos)
        h = _add_norm(self.norm_in[0], h, self.drop_h[0](self.proj_o[0](a)), self.fused)
        # Part II: attention to memory (attention.py:144-168)
        n = h.size(0)
        n_q = csr_inter[1][0].numel() - 1                  # rows of the inter graph's in-CSR
        if n_q < n:
            raise ValueError("the inter graph has fewer destination nodes than the block has states")
        hq = h if n_q == n else torch.cat([h, h.new_zeros(n_q - n, h.size(1))], 0)        # attention.py:148-149
        a = self._attend(1, heads(self.proj_q[1], hq), heads(self.proj_k[1], mem), heads(self.proj_v[1], mem), csr_inter)[:n]
        h = _add_norm(self.norm_in[1], h, self.drop_h[1](self.proj_o[1](a)), self.fused)
        # FFN (attention.py:170-171)
        return _add_norm(self.norm_inter, h, self.ffn(h), self.fused)
