"""Codebook lookup with scaling, and its gradient by sorted labels (no counterpart in the
reference).

lookup(C, labels) replaces labels by the codebook's rows: points by their centers (vector
quantisation), tokens by their embeddings.  Its gradient in C sums the rows of each label,
the center update's sum without the mean, in float32 (float64 for float64 rows) in row
order, so that it is the same on every run.
"""
import torch

import _ops
from _lib import call_on, lib, workspace
from row_groups import check_groups, group_rows


def _lookup(C, labels, scale):
    _ops.refuse_tangents(C)
    _ops.check_input(C, "C")
    rt = _ops.row_type(C, "C")
    if C.dim() != 2:
        raise RuntimeError("C must be 2D")
    i64 = _ops.check_labels(labels)
    _ops.check_same_device(labels, "labels", C, "C")
    k, d = C.shape
    out = C.new_empty((*labels.shape, d))
    call_on(C, lib().euc_codebook_lookup, rt, C.data_ptr(), k, labels.data_ptr(), i64, labels.numel(), d, scale,
            out.data_ptr())
    return out


def lookup_grad(G, labels, n_clusters, scale=1.0, groups=None):
    """grad_C [n_clusters, dim] in G's type: scale * the sum of G's rows with each label
    (G has the labels' shape and then dim; labels outside [0, n_clusters) add nothing, a
    label without rows gets zeros).  `groups`: the labels' group_rows, if the caller has it."""
    _ops.refuse_tangents(G)
    _ops.check_input(G, "G")
    rt = _ops.row_type(G, "G")
    _ops.check_labels(labels)
    k, n = int(n_clusters), labels.numel()
    if G.dim() < 1 or tuple(G.shape[:-1]) != tuple(labels.shape):
        raise RuntimeError("G must have the labels' shape and one more dimension")
    _ops.check_same_device(labels, "labels", G, "G")
    if groups is None:
        groups = group_rows(labels.reshape(-1), k)
    else:
        rows, picks, clusters = check_groups(groups)
        if clusters != k or rows * picks != n:
            raise RuntimeError("groups do not belong to these labels")
        _ops.check_same_device(groups.order, "groups", G, "G")
    d = G.size(-1)
    out = G.new_empty((k, d))
    ws = workspace(lib().euc_codebook_grad_workspace_bytes(rt, n, d), G.device)
    call_on(G, lib().euc_codebook_grad, rt, G.data_ptr(), groups.offsets.data_ptr(), groups.order.data_ptr(),
            groups.labels.data_ptr(), n, k, d, float(scale), out.data_ptr(), ws.data_ptr(), ws.numel())
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, C, labels, scale):
        ctx.save_for_backward(labels)
        ctx.k, ctx.scale = C.size(0), scale
        return _lookup(C, labels, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (labels,) = ctx.saved_tensors
        return lookup_grad(g.contiguous(), labels, ctx.k, ctx.scale), None, None


def lookup(C, labels, scale=1.0):
    """scale * C[labels] (C [k, dim] contiguous; labels int64 or int32 of any shape): the
    labels' shape and then dim, in C's type (formed in float32, float64 for
    float64, and rounded); a zero row where a label is
    outside [0, k).  Differentiable in C."""
    if isinstance(C, torch.Tensor) and C.requires_grad and torch.is_grad_enabled():
        return _Lookup.apply(C, labels, float(scale))
    return _lookup(C, labels, float(scale))
