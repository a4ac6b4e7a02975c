"""Propagation layers with the reference's call signatures.

DGLLayer.forward(graph, u_f, v_f)  -- DiffGraph-Rec/Model.py:142-174
UUGCNLayer.forward(graph, u_f)     -- DiffGraph_NC/Model.py:184-214

`graph` is a diffgraph_amd.CSRGraph instead of a dgl.DGLGraph.  The reference only ever
instantiates these with weight=False (Model.py:30), so the u_w/v_w projections are not
provided; asking for them raises.

embedding(table, ids) / Embedding  -- rows of a table by id, scaled, with the table's gradient formed by sorted tokens:
                                      the batch gathers of DiffGraph-Rec/Model.py:101-105 for tables of any width.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import ops
from .graph import CSRGraph


def _slope_of(activation) -> float:
    if activation is None:
        return 1.0
    if isinstance(activation, nn.LeakyReLU):
        return float(activation.negative_slope)
    raise NotImplementedError("only LeakyReLU (or no activation) is fused into the propagation kernel")


class DGLLayer(nn.Module):
    def __init__(self, in_feats, out_feats, weight=False, bias=False, activation=None):
        super().__init__()
        if weight or bias:
            raise NotImplementedError("the reference never enables weight/bias on its propagation layers")
        self._in_feats, self._out_feats = in_feats, out_feats
        self.weight, self.bias = weight, bias
        self._activation = activation

    def forward(self, graph: CSRGraph, u_f: torch.Tensor, v_f: torch.Tensor) -> torch.Tensor:
        node_f = torch.cat([u_f, v_f], dim=0)
        return ops.spmm_norm_act(graph, node_f, _slope_of(self._activation))


class UUGCNLayer(nn.Module):
    def __init__(self, in_feats, out_feats, weight=False, bias=False, activation=None):
        super().__init__()
        if weight or bias:
            raise NotImplementedError("the reference never enables weight/bias on its propagation layers")
        self._in_feats, self._out_feats = in_feats, out_feats
        self.weight, self.bias = weight, bias
        self._activation = activation

    def forward(self, graph: CSRGraph, u_f: torch.Tensor) -> torch.Tensor:
        return ops.spmm_norm_act(graph, u_f.contiguous(), _slope_of(self._activation))


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.consts = (table.shape[0], scale, padding_idx)
        return ops.embedding_lookup(table, ids, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        (ids,) = ctx.saved_tensors
        n_rows, scale, padding_idx = ctx.consts
        return ops.embedding_grad(d_out, ids, n_rows, scale, padding_idx), None, None, None


def embedding(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * table[ids], [*ids.shape, width], differentiable in the table (once).  Rows of ids equal to padding_idx are
    looked up like any other and get no gradient; an id outside the table gives a row of NaN and no gradient."""
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise ops.DiffGraphHipError(f"padding_idx must lie in [0,{table.shape[0]}); got {padding_idx}")
    return _EmbeddingFn.apply(table, ids, float(scale), padding_idx)


class Embedding(nn.Module):
    """A [rows, width] table (xavier_uniform_, as Model.py:45-52; a padding row starts as zeros) and its lookup."""

    def __init__(self, rows: int, width: int, scale: float = 1.0, padding_idx: Optional[int] = None, device="cuda", dtype=torch.float32):
        super().__init__()
        self.scale, self.padding_idx = float(scale), padding_idx
        if padding_idx is not None and not 0 <= padding_idx < rows:
            raise ops.DiffGraphHipError(f"padding_idx must lie in [0,{rows}); got {padding_idx}")
        table = nn.init.xavier_uniform_(torch.empty(rows, width, device=device, dtype=torch.float32))
        if padding_idx is not None:
            table[padding_idx] = 0
        self.weight = nn.Parameter(table.to(dtype))

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding(self.weight, ids, self.scale, self.padding_idx)
