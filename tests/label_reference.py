"""The label operators from their definitions in 64 bits (numpy), and the bounds that their
32-bit arithmetic stays within, for the tests of label_scores, row_groups and codebook.

u = 2^-24 is half a step of fp32.  A sum of t products of fp32 values is off by at most
(t + 1) u times the sum of the products' magnitudes, in any order; rounding a result to its
type adds at most eps / 2 of it, or half the type's smallest step where it is subnormal.
"""
import math

import numpy as np
import torch

U32, U64 = 2.0 ** -24, 2.0 ** -53


def unit(dtype):
    return U64 if dtype == torch.float64 else U32


def rounding(dtype, ref):
    """Half a step of `dtype` at the values `ref`."""
    f = torch.finfo(dtype)
    return np.maximum(np.abs(ref) * (f.eps / 2), f.smallest_normal * f.eps / 2)


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def close(got, ref, tol, what=""):
    """|got - ref| <= tol where ref is finite; the same infinities and NaN elsewhere."""
    got = f64(got) if isinstance(got, torch.Tensor) else got
    fine = np.isfinite(ref)
    assert got.shape == ref.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what + ": NaN"
    other = ~fine & ~np.isnan(ref)
    assert np.array_equal(got[other], ref[other]), what + ": infinities"
    tol = np.broadcast_to(tol, ref.shape)
    off = np.abs(got[fine] - ref[fine])
    bad = ~(off <= tol[fine])
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {off[bad].max()} over {tol[fine][bad].min()}"


def label_scores(scores, labels, scale, top):
    """(log_probs or None, entropy, top_log_probs, top_labels, p, log_p) in 64 bits."""
    with np.errstate(all="ignore"):
        x = f64(scores)
        y = x * math.copysign(1.0, scale)
        n, m = x.shape
        hi = y.max(1) if n else np.zeros(0)          # NaN where the row holds one
        empty = hi == -np.inf
        d = (y - np.where(empty, 0.0, hi)[:, None]) * abs(scale)
        e = np.exp(d)
        S = e.sum(1)
        L = np.where(empty, -np.inf, np.log(S))
        bad = np.isnan(hi) | (hi == np.inf)
        log_p = d - np.where(empty, 0.0, L)[:, None]
        log_p[bad] = np.nan
        p = np.exp(log_p)
        p[empty] = 0.0
        H = -np.where(p > 0, p * log_p, 0.0 * p).sum(1)
        log_p[empty] = -np.inf
        # NaN first, then larger first, then the lower index
        key = np.where(np.isnan(y), np.inf, y)
        order = np.lexsort((np.broadcast_to(np.arange(m), y.shape), -key, ~np.isnan(y)), axis=1)[:, :top]
        lp = None
        if labels is not None:
            lab = labels.cpu().numpy()
            ok = (lab >= 0) & (lab < m)
            lp = np.where(ok, log_p[np.arange(n), np.where(ok, lab, 0)], 0.0)
        return lp, H, np.take_along_axis(log_p, order, 1), order, p, log_p


def score_bounds(m, dtype, log_p):
    """(of L, of the entropy, of a log probability).  A term exp(d) is off by a factor within
    (3 + 2.4 |d|) 2u: d by u of a subtraction and of a multiplication, and the exponential by
    2 + 1.16 |d| steps of 2u.  S weighs these with p, E_p |d| <= log m, plus m / 128 + 24
    additions; T likewise with p |d|, E_p d^2 <= (log m + 2)^2."""
    u, lm = unit(dtype), math.log(m) + 2.0
    adds = m / 128 + 24
    tL = u * (2 * (3 + 2.4 * lm) + adds + 2 * lm)
    tH = tL + u * lm * (2 * (4 + 2.4 * lm) + 2 * adds + 4)
    mag = np.where(np.isfinite(log_p), np.abs(log_p), 0.0)
    return tL, tH, tL + u * 4 * (mag + lm)


def label_scores_grad(p, log_p, H, labels, scale, gl, ge, dtype):
    """(gradient, bound) with rows of nothing left zero."""
    n, m = p.shape
    u = unit(dtype)
    with np.errstate(all="ignore"):
        empty = (p == 0).all(1)
        lab = labels.cpu().numpy() if labels is not None else np.full(n, -1)
        ok = (lab >= 0) & (lab < m)
        gl = np.where(ok, f64(gl), 0.0) if gl is not None else np.zeros(n)
        ge = f64(ge) if ge is not None else np.zeros(n)
        hit = np.zeros((n, m))
        hit[np.arange(n)[ok], lab[ok]] = 1.0
        lp0 = np.where(p > 0, log_p, 0.0)
        inner = gl[:, None] + ge[:, None] * (lp0 + H[:, None])
        ref = scale * (gl[:, None] * hit - np.where(p > 0, p * inner, 0.0 * p))
        ref[empty] = 0.0
        tL, tH, tp = score_bounds(m, dtype, np.where(p > 0, log_p, 0.0))
        size = np.abs(gl)[:, None] + np.abs(ge)[:, None] * (np.abs(lp0) + H[:, None])
        rel = tp + (2 + 1.16 * np.abs(lp0)) * 2 * u + 8 * u
        tol = abs(scale) * (p * (rel * size + np.abs(ge)[:, None] * (tp + tH)) + 4 * u * np.abs(gl)[:, None] * hit)
        # below the smallest normal the exponential is flushed to zero
        tol += abs(scale) * size * torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).tiny * 4
    return ref, tol + rounding(dtype, ref)


def group_rows(labels, k):
    """(offsets, order, position, labels) with the definition's stable order."""
    flat = labels.cpu().numpy().reshape(-1).astype(np.int64)
    keep = np.nonzero((flat >= 0) & (flat < k))[0]
    order = keep[np.argsort(flat[keep], kind="stable")]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[keep], minlength=k)[:k])])
    full = np.full(flat.size, -1, dtype=np.int64)
    full[:order.size] = order
    pos = np.full(flat.size, -1, dtype=np.int64)
    pos[order] = np.arange(order.size)
    lab = np.full(flat.size, -1, dtype=np.int64)
    lab[:order.size] = flat[order]
    return offsets, full, pos.reshape(labels.shape), lab
