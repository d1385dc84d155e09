"""Calls of the label operators at the edges of what they take: the sort's passes in one block
and in tiles up to the largest number of labels, rows alone and among others, the posterior in
blocks of rows, NaN where nothing is read, and gradients captured into a graph."""
import math

import numpy as np
import pytest
import torch

import _ops
import label_reference as ref
from codebook import lookup, lookup_grad
from kmeans import LloydKMeans
from label_scores import label_log_probs, label_log_probs_grad
from row_groups import group_rows, rows_from_groups, rows_from_groups_grad, rows_to_groups

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# keys of 12, 23, 29 and 31 bits: two passes and three, in one block up to 1024 slots
@pytest.mark.parametrize("k", [2049, 5000, 2 ** 22, 2 ** 28, 2 ** 31 - 2])
@pytest.mark.parametrize("n", [1, 33, 1000, 1024, 1025, 5000])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_sort_of_far_labels(n, k, dtype):
    """With k = 2^31 - 2 the offsets take 8 GiB."""
    lab = torch.randint(0, k, (n,), generator=gen(n), device="cuda")
    lab[n // 2:] = lab[n // 2:] % 7 + k - 7  # equal ones, at the far end
    lab[::5] = torch.where(lab[::5] % 2 == 0, -1 - lab[::5] % 3, torch.full_like(lab[::5], 2 ** 31 - 1))
    lab[0] = k - 1
    lab = lab.to(dtype)
    got = group_rows(lab, k)
    flat = lab.long().cpu().numpy()
    keep = np.nonzero((flat >= 0) & (flat < k))[0]
    order = keep[np.argsort(flat[keep], kind="stable")]
    full, pos = np.full(n, -1), np.full(n, -1)
    full[:order.size] = order
    pos[order] = np.arange(order.size)
    assert np.array_equal(got.order.cpu().numpy(), full)
    assert np.array_equal(got.position.cpu().numpy(), pos)
    assert np.array_equal(got.labels.cpu().numpy(), np.where(full >= 0, flat[full], -1))
    assert got.offsets.numel() == k + 1
    at = np.unique(np.concatenate([flat[order], flat[order] + 1, [0, k // 2, k - 1, k]]))
    want = np.searchsorted(flat[order], at)
    assert np.array_equal(got.offsets[torch.from_numpy(at).cuda()].cpu().numpy(), want)


@pytest.mark.parametrize("n,m", [(1000, 40000), (600, 40000), (1000, 3000), (3000, 1500), (500, 131072)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_row_alone_and_among_others(n, m, dtype):
    """The kernel, its block size and its clusters go by the number of rows, so the sums' last
    bits may differ; both stay within the bound, and the alternatives are the same."""
    x = (torch.randn(n, m, generator=gen(m), device="cuda") * 3).to(dtype)
    lab = torch.randint(0, m, (n,), generator=gen(n), device="cuda")
    many = label_log_probs(x, lab, 0.7, 8)
    for i in (0, n // 2, n - 1):
        rows = slice(i, i + 1)
        lp, H, tlp, tl, _, log_p = ref.label_scores(x[rows], lab[rows], 0.7, 8)
        _, tH, tp = ref.score_bounds(m, dtype, log_p)
        for r, at in ((many, rows), (label_log_probs(x[rows], lab[rows], 0.7, 8), slice(0, 1))):
            ref.close(r.log_probs[at], lp, tp[[0], lab[rows].cpu().numpy()], "log_probs")
            ref.close(r.entropy[at], H, tH, "entropy")
            ref.close(r.top_log_probs[at], tlp, np.take_along_axis(tp, tl, 1), "top_log_probs")
            assert np.array_equal(r.top_labels[at].cpu().numpy(), tl)


@pytest.mark.parametrize("op", ["fp16_fp32", "single", "double"])
def test_posterior_of_many_centers_in_blocks(op):
    """3000 centers, a short last block: each row from its block's distances."""
    dt = torch.float64 if op == "double" else torch.float32
    C = torch.randn(3000, 24, generator=gen(1), device="cuda", dtype=dt)
    X = C[:700] + 0.3 * torch.randn(700, 24, generator=gen(2), device="cuda", dtype=dt)
    lab = torch.arange(700, device="cuda").to(torch.int32)
    km = LloydKMeans(3000, op=op, kappa=0.5)
    for rows in (None, 640, 333):
        r = km.posterior(X, C, temperature=0.5, labels=lab, top=5, block_rows=rows)
        D = torch.cat([_ops.run_distance(op, X[lo:lo + (rows or 700)], C, 0.5) for lo in range(0, 700, rows or 700)])
        lp, H, tlp, tl, _, log_p = ref.label_scores(D, lab, -2.0, 5)
        _, tH, tp = ref.score_bounds(3000, D.dtype, log_p)
        ref.close(r.log_probs, lp, tp[np.arange(700), np.arange(700)], "log_probs")
        ref.close(r.entropy, H, tH, "entropy")
        ref.close(r.top_log_probs, tlp, np.take_along_axis(tp, tl, 1), "top_log_probs")
        assert np.array_equal(r.top_labels.cpu().numpy(), tl)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [7, 64, 333])
def test_nan_where_nothing_is_read(d, dtype):
    """Rows behind the last kept slot, weights of dropped picks and gradient rows of dropped
    labels hold NaN; nothing of it arrives."""
    n, p, k = 300, 3, 11
    lab = torch.randint(-3, k + 3, (n, p), generator=gen(d), device="cuda")
    groups = group_rows(lab, k)
    kept = int(groups.offsets[-1])
    dropped = (lab < 0) | (lab >= k)
    Y = torch.randn(n * p, d, generator=gen(1), device="cuda").to(dtype)
    G = torch.randn(n, d, generator=gen(2), device="cuda").to(dtype)
    W = torch.rand(n, p, generator=gen(3), device="cuda")
    clean = (rows_from_groups(Y, groups, W), *rows_from_groups_grad(G, Y, groups, W), rows_from_groups(Y, groups))
    Y[kept:] = math.nan
    W[dropped] = math.nan
    dirty = (rows_from_groups(Y, groups, W), *rows_from_groups_grad(G, Y, groups, W), rows_from_groups(Y, groups))
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))
    rows = torch.randn(n, p, d, generator=gen(4), device="cuda").to(dtype)
    want = lookup_grad(rows, lab, k)
    rows[dropped] = math.nan
    assert torch.equal(lookup_grad(rows, lab, k), want)


def test_gradients_captured_into_a_graph():
    """Forward and gradients of a whole step (points to their 2 likeliest centers, the residuals
    there and back) in one graph, replayed over other inputs; no eager graph of the same leaves
    is alive meanwhile."""
    n, k, d, p = 200, 30, 40, 2
    X, C, L = (torch.zeros(*s, device="cuda", requires_grad=True) for s in ((n, d), (k, d), (n, k)))
    W = torch.zeros(n, p, device="cuda", requires_grad=True)
    G = torch.randn(n, d, generator=gen(9), device="cuda")

    def step():
        r = label_log_probs(L, None, 0.5, p)
        groups = group_rows(r.top_labels, k)
        Y = rows_to_groups(X, groups) - lookup(C, groups.labels)
        out = rows_from_groups(Y, groups, W)
        return (out.detach(), *torch.autograd.grad((out * G).sum() + r.entropy.sum(), (X, C, L, W)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        with torch.no_grad():
            for t in (X, C, L, W):
                t.copy_(torch.randn(t.shape, generator=gen(seed + t.numel()), device="cuda"))
        graph.replay()
        kept = [t.clone() for t in got]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
        assert all(float(t.abs().max()) > 0 for t in want)


def test_rows_of_a_wide_buffer_beginning_anywhere():
    """Scores that are columns of a wider buffer, beginning anywhere: the gradient is contiguous."""
    buf = torch.randn(9, 5000, generator=gen(1), device="cuda").bfloat16()
    lab = torch.arange(9, device="cuda").to(torch.int32)
    one = torch.ones(9, device="cuda")
    for lo, m in ((0, 4999), (1, 4096), (3, 777), (7, 64), (13, 1)):
        x = buf[:, lo:lo + m]
        r, same = label_log_probs(x, lab, 1.0, min(m, 5)), label_log_probs(x.contiguous(), lab, 1.0, min(m, 5))
        assert torch.equal(r.top_labels, same.top_labels)
        g = label_log_probs_grad(x, lab, r.row_stats, one, one)
        assert torch.equal(g, label_log_probs_grad(x.contiguous(), lab, r.row_stats, one, one))
