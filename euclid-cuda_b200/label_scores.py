"""Log probabilities of rows of scores: of given labels, with the entropy and the best
alternatives, and their gradient (no counterpart in the reference).

A score is a squared distance from any of the distance operators (scale = -1 /
temperature: the soft assignment of points to centers) or any other logit.  With
z = scale * scores, log p_j = z_j - log sum exp z; a score with z = -inf is masked.  The
argmin operators give a row's label; these give how sure it is.
"""
from typing import NamedTuple, Optional

import torch

import _ops
from _lib import call_on, lib

MAX_TOP = 32


class LabelLogProbs(NamedTuple):
    """Per row, in float32 (float64 for float64 scores): the given label's log probability
    (None without labels; 0 where the label is outside the columns), the entropy, the
    `top` best labels (int64) with their log probabilities, and what the gradient needs
    (largest score, log of the sum, entropy)."""
    log_probs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_log_probs: torch.Tensor
    top_labels: torch.Tensor
    row_stats: torch.Tensor


def _check(scores, labels, scale):
    if not isinstance(scores, torch.Tensor):
        raise TypeError("scores must be a torch.Tensor")
    _ops.refuse_tangents(scores)
    if not scores.is_cuda:
        raise RuntimeError("scores must be a CUDA tensor")
    if scores.dim() != 2:
        raise RuntimeError("scores must be 2D")
    n, m = scores.shape
    if m < 1:
        raise RuntimeError("scores must have at least one column")
    if (m > 1 and scores.stride(1) != 1) or (n > 1 and scores.stride(0) < m):
        raise RuntimeError("rows of scores must be contiguous and must not overlap")
    rt = _ops.row_type(scores, "scores")
    i64 = 1
    if labels is not None:
        i64 = _ops.check_labels(labels)
        if tuple(labels.shape) != (n,):
            raise RuntimeError(f"labels must have shape {(n,)}")
        _ops.check_same_device(labels, "labels", scores, "scores")
    if not (0.0 < abs(scale) < float("inf")):
        raise RuntimeError("scale must be finite and not 0")
    return n, m, max(scores.stride(0), m), rt, i64


def _forward(scores, labels, scale, top):
    n, m, ld, rt, i64 = _check(scores, labels, scale)
    if not 0 <= top <= min(m, MAX_TOP):
        raise RuntimeError(f"top must be in [0, min(columns, {MAX_TOP})]")
    new, acc = scores.new_empty, _ops.acc_dtype(scores)  # (2 us less a call than torch.empty)
    log_probs = new(n, dtype=acc) if labels is not None else None
    entropy = new(n, dtype=acc)
    stats = new((n, 3), dtype=acc)
    top_lp = new((n, top), dtype=acc)
    top_lab = new((n, top), dtype=torch.int64)
    call_on(scores, lib().euc_label_log_probs, rt, scores.data_ptr(), ld, n, m,
            labels.data_ptr() if labels is not None else None, i64, scale, top,
            log_probs.data_ptr() if labels is not None else None, entropy.data_ptr(), stats.data_ptr(),
            top_lp.data_ptr(), top_lab.data_ptr())
    return LabelLogProbs(log_probs, entropy, top_lp, top_lab, stats)


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, labels, scale, top):
        r = _forward(scores, labels, scale, top)
        ctx.save_for_backward(scores, labels, r.row_stats)
        ctx.scale = scale
        ctx.set_materialize_grads(False)  # an output that the loss leaves out costs nothing
        ctx.mark_non_differentiable(r.top_log_probs, r.top_labels, r.row_stats)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_log_probs, g_entropy, *_):
        scores, labels, stats = ctx.saved_tensors
        if g_log_probs is None and g_entropy is None:
            return None, None, None, None
        g = label_log_probs_grad(scores, labels, stats,
                                 g_log_probs.contiguous() if g_log_probs is not None else None,
                                 g_entropy.contiguous() if g_entropy is not None else None, ctx.scale)
        return g, None, None, None


def label_log_probs(scores, labels=None, scale=1.0, top=0):
    """LabelLogProbs of scores (n x m, CUDA; rows contiguous, their stride free) for the
    labels (int64 or int32 [n], optional).  `top` (at most 32) alternatives by scale *
    scores, equal ones by the lower index.  A row with every score masked has log
    probabilities of -inf and entropy 0; a row with a NaN or scale * score = +inf has NaN.
    |scale| is at least 2^-120 (float16 2^-126, float64 2^-1014), at most 2^126 (float64 2^1022).
    Differentiable in scores through log_probs and entropy (not through the alternatives)."""
    scale, top = float(scale), int(top)
    if isinstance(scores, torch.Tensor) and scores.requires_grad and torch.is_grad_enabled():
        return LabelLogProbs(*_LogProbs.apply(scores, labels, scale, top))
    return _forward(scores, labels, scale, top)


def label_log_probs_grad(scores, labels, row_stats, grad_log_probs=None, grad_entropy=None, scale=1.0):
    """The gradient, in the scores' type (n x m, contiguous), of sum(grad_log_probs *
    log_probs + grad_entropy * entropy) with respect to the scores; `row_stats` is the
    forward call's.  Either gradient may be None; labels are needed with grad_log_probs."""
    scale = float(scale)
    n, m, ld, rt, i64 = _check(scores, labels, scale)
    _ops.refuse_tangents(grad_log_probs, grad_entropy)
    acc = _ops.acc_dtype(scores)
    _ops.check_like(row_stats, "row_stats", (n, 3), acc, scores.device)
    if grad_log_probs is not None:
        if labels is None:
            raise RuntimeError("grad_log_probs needs labels")
        _ops.check_like(grad_log_probs, "grad_log_probs", (n,), acc, scores.device)
    if grad_entropy is not None:
        _ops.check_like(grad_entropy, "grad_entropy", (n,), acc, scores.device)
    grad = scores.new_empty((n, m))
    call_on(scores, lib().euc_label_log_probs_grad, rt, scores.data_ptr(), ld, n, m,
            labels.data_ptr() if labels is not None else None, i64, scale, row_stats.data_ptr(),
            grad_log_probs.data_ptr() if grad_log_probs is not None else None,
            grad_entropy.data_ptr() if grad_entropy is not None else None, grad.data_ptr())
    return grad
