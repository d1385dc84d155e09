"""Rows sorted by label and back, with weights applied, and their gradients (no counterpart
in the reference; the center update sorts its rows by label internally).

Rows go to the clusters that their labels name (one label a row, or several picks), are
contiguous per cluster there, and come back as weighted sums:

    groups = group_rows(labels, n_clusters)          # labels [n] or [n, picks]
    Y = rows_to_groups(X, groups)                    # rows of cluster c: Y[offsets[c]:offsets[c + 1]]
    out = rows_from_groups(f(Y), groups, weights)    # out[i] = sum_j weights[i, j] f(Y)[position[i, j]]

The sort is stable and nothing depends on the order of atomics, so every result is the same
on every run.  Nothing waits for the device: Y has n * picks rows whatever was dropped.
"""
from typing import NamedTuple

import torch

import _ops
from _lib import call_on, lib, workspace


class RowGroups(NamedTuple):
    """offsets [n_clusters + 1]: first sorted position of each cluster, and the number of
    slots kept; order [n * picks]: slot (row * picks + pick) at each sorted position, -1
    behind the last; position (the labels' shape): sorted position of each slot, -1 where
    its label is outside [0, n_clusters); labels [n * picks]: label at each sorted
    position, -1 behind the last.  All int32."""
    offsets: torch.Tensor
    order: torch.Tensor
    position: torch.Tensor
    labels: torch.Tensor

    @property
    def n_clusters(self):
        return self.offsets.numel() - 1

    @property
    def n_rows(self):
        return self.position.size(0)

    @property
    def picks(self):
        return self.position.size(1) if self.position.dim() == 2 else 1


def group_rows(labels, n_clusters):
    """RowGroups of labels (int64 or int32, [n] or [n, picks], CUDA): slots of one label in
    slot order; labels outside [0, n_clusters) are dropped, as by update_centers_*."""
    i64 = _ops.check_labels(labels)
    if labels.dim() not in (1, 2):
        raise RuntimeError("labels must be 1D or 2D")
    k, slots, new = int(n_clusters), labels.numel(), labels.new_empty
    if k < 0 or k > 2 ** 31 - 2 or slots > 2 ** 31 - 2:
        raise RuntimeError("n_clusters and the number of labels must be in [0, 2^31 - 2]")
    offsets = new(k + 1, dtype=torch.int32)
    order = new(slots, dtype=torch.int32)
    position = new(labels.shape, dtype=torch.int32)
    sorted_labels = new(slots, dtype=torch.int32)
    need = lib().euc_group_rows_workspace_bytes(slots, k)
    ws = workspace(need, labels.device) if need else None
    call_on(labels, lib().euc_group_rows, labels.data_ptr(), i64, slots, k, offsets.data_ptr(), order.data_ptr(),
            position.data_ptr(), sorted_labels.data_ptr(), ws.data_ptr() if need else None, need)
    return RowGroups(offsets, order, position, sorted_labels)


def check_groups(groups):
    """A RowGroups whose parts fit together (their values are checked by the kernels):
    (rows, picks, clusters)."""
    if not isinstance(groups, RowGroups):
        raise TypeError("groups must be a RowGroups")
    offsets, order, position, labels = groups
    for t, name in ((offsets, "offsets"), (order, "order"), (position, "position"), (labels, "labels")):
        _ops.check_input(t, name)
        if t.dtype != torch.int32 or t.get_device() != offsets.get_device():
            raise RuntimeError(f"groups.{name} must be int32 on the groups' device")
    slots, shape = position.numel(), position.shape
    if offsets.dim() != 1 or offsets.numel() < 1 or len(shape) not in (1, 2) or \
            order.numel() != slots or labels.numel() != slots:
        raise RuntimeError("groups do not fit together")
    return shape[0], shape[1] if len(shape) == 2 else 1, offsets.numel() - 1


def _check_rows(t, name, rows, groups):
    _ops.check_input(t, name)
    rt = _ops.row_type(t, name)
    if t.dim() != 2 or t.size(0) != rows:
        raise RuntimeError(f"{name} must be 2D with {rows} rows")
    _ops.check_same_device(t, name, groups.position, "groups")
    return rt, t.size(1)


def _kept(groups, k):
    return groups.offsets.data_ptr() + 4 * k


def _to_groups(X, groups):
    _ops.refuse_tangents(X)
    n, p, k = check_groups(groups)
    rt, d = _check_rows(X, "X", n, groups)
    Y = X.new_empty((n * p, d))
    call_on(X, lib().euc_rows_to_groups, rt, X.data_ptr(), groups.position.data_ptr(), _kept(groups, k), n, p, d,
            Y.data_ptr())
    return Y


def _check_weights(weights, Y, groups):
    if weights is not None:
        _ops.check_like(weights, "weights", groups.position.shape, _ops.acc_dtype(Y), Y.device)


def _from_groups(Y, groups, weights):
    _ops.refuse_tangents(Y, weights)
    n, p, _ = check_groups(groups)
    rt, d = _check_rows(Y, "Y", n * p, groups)
    _check_weights(weights, Y, groups)
    out = Y.new_empty((n, d))
    call_on(Y, lib().euc_rows_from_groups, rt, Y.data_ptr(), groups.position.data_ptr(),
            weights.data_ptr() if weights is not None else None, n, p, d, out.data_ptr())
    return out


def rows_from_groups_grad(grad_out, Y, groups, weights=None):
    """Gradients of rows_from_groups: (grad_Y, grad_weights), the second None without
    weights.  grad_Y[position[i, j]] = weights[i, j] * grad_out[i], zero rows behind the
    last kept slot; grad_weights[i, j] = <grad_out[i], Y[position[i, j]]>, 0 where dropped."""
    n, p, _ = check_groups(groups)
    _, d = _check_rows(Y, "Y", n * p, groups)
    _check_weights(weights, Y, groups)
    _ops.check_like(grad_out, "grad_out", (n, d), Y.dtype, Y.device)
    return _from_groups_grad(grad_out, Y, groups, weights, True, weights is not None)


def _from_groups_grad(grad_out, Y, groups, weights, want_Y, want_weights):
    """The wanted ones of (grad_Y, grad_weights), None for the other; grad_Y needs the
    weights (None for ones), grad_weights needs Y."""
    _ops.refuse_tangents(grad_out, Y, weights)
    n, p, k = check_groups(groups)
    rt, d = _check_rows(grad_out, "grad_out", n, groups)
    grad_Y = grad_out.new_empty((n * p, d)) if want_Y else None
    grad_w = grad_out.new_empty(groups.position.shape, dtype=_ops.acc_dtype(grad_out)) if want_weights else None
    call_on(grad_out, lib().euc_rows_from_groups_grad, rt, grad_out.data_ptr(),
            Y.data_ptr() if want_weights else None, groups.position.data_ptr(),
            weights.data_ptr() if weights is not None else None, _kept(groups, k), n, p, d,
            grad_Y.data_ptr() if want_Y else None, grad_w.data_ptr() if want_weights else None)
    return grad_Y, grad_w


class _ToGroups(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, groups):
        Y = _to_groups(X, groups)
        ctx.save_for_backward(*groups)  # (refuses a backward pass after a change in place)
        return Y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return _from_groups(g.contiguous(), RowGroups(*ctx.saved_tensors), None), None


class _FromGroups(torch.autograd.Function):
    @staticmethod
    def forward(ctx, Y, groups, weights):
        out = _from_groups(Y, groups, weights)
        # each gradient needs the other input: Y, the largest tensor, is kept for the weights' alone
        need_Y, _, need_weights = ctx.needs_input_grad
        ctx.save_for_backward(Y if need_weights else None, weights if need_Y else None, *groups)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        Y, weights, *groups = ctx.saved_tensors
        need_Y, _, need_weights = ctx.needs_input_grad
        grad_Y, grad_w = _from_groups_grad(g.contiguous(), Y, RowGroups(*groups), weights, need_Y, need_weights)
        return grad_Y, None, grad_w


def rows_to_groups(X, groups):
    """Y [n * picks, dim] with Y[position[i, j]] = X[i] (X [n, dim], contiguous): the rows of
    cluster c are Y[offsets[c]:offsets[c + 1]]; rows behind the last kept slot are zero.
    Differentiable in X."""
    if isinstance(X, torch.Tensor) and X.requires_grad and torch.is_grad_enabled():
        return _ToGroups.apply(X, groups)
    return _to_groups(X, groups)


def rows_from_groups(Y, groups, weights=None):
    """out [n, dim] with out[i] = sum over the kept picks j, in order, of weights[i, j] *
    Y[position[i, j]] (weights float32, float64 for float64 rows, of the labels' shape;
    None for ones), summed in float32 (float64) and rounded once.  Differentiable in Y and
    weights."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (Y, weights)):
        return _FromGroups.apply(Y, groups, weights)
    return _from_groups(Y, groups, weights)
