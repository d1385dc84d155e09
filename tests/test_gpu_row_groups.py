"""group_rows, rows_to_groups, rows_from_groups and the gradients against their definitions:
the stable order exactly, the rows there exactly, the sums within their derived bounds."""
import threading

import numpy as np
import pytest
import torch

import label_reference as ref
from row_groups import RowGroups, group_rows, rows_from_groups, rows_from_groups_grad, rows_to_groups

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_labels(shape, k, seed, kind="even"):
    g = gen(seed)
    if kind == "one":  # every slot in one cluster
        return torch.full(shape, max(0, k - 1), device="cuda", dtype=torch.int64)
    if kind == "none":  # every slot dropped
        return torch.full(shape, k, device="cuda", dtype=torch.int64)
    if kind == "skew":
        u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
        return ((k + 1.0) ** u - 1).long().clamp_(0, k - 1)
    lab = torch.randint(0, max(1, k), shape, generator=g, device="cuda")
    if kind == "drop":
        r = torch.rand(shape, generator=g, device="cuda")
        lab = torch.where(r < 0.1, -7, torch.where(r > 0.8, k + 3, lab))
    return lab


def check_sort(labels, k):
    got = group_rows(labels, k)
    for g, w, name in zip(got, ref.group_rows(labels, k), RowGroups._fields):
        assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), w), name
    return got


@pytest.mark.parametrize("kind", ["even", "drop", "one", "none", "skew"])
@pytest.mark.parametrize("n,k", [(1, 1), (31, 2), (33, 64), (4095, 37), (4096, 1024), (4097, 4096), (20000, 4095),
                                 (20000, 4097), (9000, 131072), (70000, 9), (300000, 1000), (270000, 70000)])
def test_sort(n, k, kind):
    check_sort(make_labels((n,), k, n + k, kind), k)


@pytest.mark.parametrize("k", [1, 5000, 20_000_000, 2 ** 31 - 2])
def test_sort_int32_and_many_labels(k):
    """int32 labels, up to three passes (with far labels, the offsets are as long as k)."""
    if k > 10 ** 8:
        k = 2 ** 28  # 29 key bits: three passes; 1 GiB of offsets
    lab = torch.randint(0, k, (5000,), generator=gen(k % 997), device="cuda").to(torch.int32)
    lab[17], lab[400] = -2 ** 31, 2 ** 31 - 1
    lab[18:40] = lab[50]
    got = group_rows(lab, k)
    flat = lab.long().cpu().numpy()
    keep = np.nonzero((flat >= 0) & (flat < k))[0]
    order = keep[np.argsort(flat[keep], kind="stable")]
    assert np.array_equal(got.order.cpu().numpy()[:order.size], order) and int(got.order[order.size:].max()) == -1
    assert np.array_equal(got.labels.cpu().numpy()[:order.size], flat[order])
    at = np.unique(np.concatenate([flat[order][::50], flat[order][::50] + 1, [0, k]]))
    want = np.searchsorted(flat[order], at)
    assert np.array_equal(got.offsets[torch.from_numpy(at).cuda()].cpu().numpy(), want)


def test_sort_of_nothing():
    g = group_rows(torch.empty(0, dtype=torch.int64, device="cuda"), 5)
    assert torch.equal(g.offsets, torch.zeros(6, dtype=torch.int32, device="cuda")) and g.order.numel() == 0
    g = group_rows(torch.zeros(7, 3, dtype=torch.int64, device="cuda"), 0)
    assert g.offsets.tolist() == [0] and int(g.position.max()) == -1 and int(g.order.max()) == -1
    X = torch.randn(7, 8, device="cuda")
    assert torch.equal(rows_to_groups(X, g), torch.zeros(21, 8, device="cuda"))
    assert torch.equal(rows_from_groups(rows_to_groups(X, g), g), torch.zeros_like(X))


def check_rows(n, p, k, d, dtype, kind, seed, make=None):
    g = gen(seed)
    lab = make_labels((n, p), k, seed, kind)
    groups = check_sort(lab, k)
    make = make or (lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float64).to(dtype))
    X, Z, G = make(n, d), make(n * p, d), make(n, d)
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    W = torch.randn(n, p, generator=g, device="cuda", dtype=acc)
    order, pos = groups.order.cpu().numpy(), groups.position.cpu().numpy()
    kept = int(groups.offsets[-1])
    Y = rows_to_groups(X, groups)
    want = np.zeros((n * p, d))
    want[:kept] = ref.f64(X)[order[:kept] // p]
    assert np.array_equal(ref.f64(Y), want)

    u = ref.unit(dtype)
    Zd, Gd, Wd = ref.f64(Z), ref.f64(G), ref.f64(W)
    here = pos >= 0
    Zp = np.where(here[:, :, None], Zd[np.where(here, pos, 0)], 0.0)  # n, p, d
    for w in (W, None):
        wd = np.where(here, Wd if w is not None else 1.0, 0.0)
        terms = wd[:, :, None] * Zp
        out = terms.sum(1)
        tol = (p + 2) * u * np.abs(terms).sum(1)
        ref.close(rows_from_groups(Z, groups, w), out, tol + ref.rounding(dtype, out), "rows_from_groups")
        gY, gW = rows_from_groups_grad(G, Z, groups, w)
        want = np.zeros((n * p, d))
        want[:kept] = (wd.reshape(-1)[order[:kept]])[:, None] * Gd[order[:kept] // p]
        ref.close(gY, want, 2 * u * np.abs(want) + ref.rounding(dtype, want), "grad_Y")
        if w is None:
            assert gW is None
        else:
            prod = Gd[:, None, :] * Zp
            ref.close(gW, np.where(here, prod.sum(2), 0.0), (d + 2) * u * np.abs(prod).sum(2), "grad_weights")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["even", "drop"])
@pytest.mark.parametrize("n,p,k,d", [(1, 1, 1, 1), (1, 4, 8, 2048), (5, 2, 3, 7), (17, 3, 64, 33), (64, 8, 16, 256),
                                     (100, 5, 7, 1001), (3, 33, 10, 96), (40, 1, 4, 4100), (9, 6, 5, 515)])
def test_rows(n, p, k, d, dtype, kind):
    check_rows(n, p, k, d, dtype, kind, seed=n * p + d)


@pytest.mark.parametrize("kind", ["one", "none", "skew"])
def test_rows_in_one_cluster_or_none(kind):
    check_rows(50, 4, 9, 128, torch.bfloat16, kind, seed=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_alignments(dtype, shift):
    """Contiguous rows that start off a 16-byte boundary."""
    g = gen(shift)

    def make(n, d):
        return torch.randn(n * d + shift, generator=g, device="cuda").to(dtype)[shift:].view(n, d)
    check_rows(12, 3, 5, 128, dtype, "drop", seed=shift, make=make)


def test_labels_of_one_dimension():
    lab = make_labels((500,), 20, 1, "drop")
    groups = check_sort(lab, 20)
    X = torch.randn(500, 16, device="cuda")
    Y = rows_to_groups(X, groups)
    kept = int(groups.offsets[-1])
    assert torch.equal(Y[:kept], X[groups.order[:kept].long()])
    back = rows_from_groups(Y, groups)
    assert torch.equal(back, torch.where((groups.position >= 0)[:, None], X, 0.0))


def test_the_same_cluster_twice_in_a_row():
    lab = torch.tensor([[2, 2, 2], [0, 2, 0]], device="cuda")
    check_sort(lab, 3)
    groups = group_rows(lab, 3)
    X = torch.randn(2, 40, device="cuda")
    assert torch.equal(rows_from_groups(rows_to_groups(X, groups), groups), (X + X) + X)


def test_gradients_against_differences():
    lab = make_labels((6, 3), 4, 8, "drop")
    groups = group_rows(lab, 4)
    g = gen(2)
    X = torch.randn(6, 5, generator=g, device="cuda", dtype=torch.float64, requires_grad=True)
    W = torch.randn(6, 3, generator=g, device="cuda", dtype=torch.float64, requires_grad=True)
    A = torch.randn(18, 5, generator=g, device="cuda", dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda x, w: rows_from_groups(rows_to_groups(x, groups) * A, groups, w), (X, W))
    assert torch.autograd.gradcheck(lambda x: rows_from_groups(rows_to_groups(x, groups), groups), (X,))


def test_broadcast_gradient():
    lab = make_labels((30, 2), 4, 8)
    groups = group_rows(lab, 4)
    X = torch.randn(30, 24, device="cuda", requires_grad=True)
    W = torch.rand(30, 2, device="cuda", requires_grad=True)
    rows_from_groups(rows_to_groups(X, groups), groups, W).sum().backward()  # a gradient of stride 0
    tol = 4 * ref.U32
    ref.close(X.grad, ref.f64(W).sum(1, keepdims=True).repeat(24, 1), tol * ref.f64(W).sum(1, keepdims=True), "X")
    ref.close(W.grad, ref.f64(X).sum(1, keepdims=True).repeat(2, 1),
              26 * ref.U32 * np.abs(ref.f64(X)).sum(1, keepdims=True), "W")


def test_far_rows():
    """Sorted rows beyond 2^31 elements."""
    n, p, d = 33000, 8, 8192  # 2.16e9 elements
    lab = torch.arange(n * p, device="cuda").view(n, p) % 64
    groups = group_rows(lab, 64)
    X = torch.randn(n, d, generator=gen(1), device="cuda").bfloat16()
    Y = rows_to_groups(X, groups)
    at = torch.tensor([0, 1, n * p // 2, n * p - 2, n * p - 1], device="cuda")
    assert torch.equal(Y[at], X[groups.order[at].long() // p])
    out = rows_from_groups(Y, groups)
    assert torch.equal(out, (8 * X.float()).bfloat16())


def test_other_stream_captured_and_repeated():
    lab = make_labels((700, 4), 50, 1, "drop")
    X = torch.randn(700, 200, generator=gen(4), device="cuda").half()
    W = torch.rand(700, 4, generator=gen(5), device="cuda")

    def chain(lab, X):
        g = group_rows(lab, 50)
        Y = rows_to_groups(X, g)
        return (*g, Y, rows_from_groups(Y, g, W), *rows_from_groups_grad(X, Y, g, W))
    want = chain(lab, X)
    assert all(torch.equal(a, b) for a, b in zip(want, chain(lab, X)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(lab, X)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    ls, Xs = torch.zeros_like(lab), torch.zeros_like(X)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = chain(ls, Xs)
        graphs.append((g, got))
    ls.copy_(lab)
    Xs.copy_(X)
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(700, 33), (700, 45), (700, 333), (12000, 33), (9000, 47), (1500, 333), (30, 16001)])
def test_odd_rows_of_16_bits(n, d, dtype):
    """Neighbouring rows share 16-byte words: what is in one reaches no other's sum."""
    check_rows(n, 6, 20, d, dtype, "drop", d)
    g = group_rows(make_labels((n, 3), 20, d, "even"), 20)
    Y = torch.randn(3 * n, d, generator=gen(d), device="cuda").to(dtype)
    bad = [0, 1, n, 3 * n - 1]
    Y[bad] = float("nan")
    out = rows_from_groups(Y, g).isnan()
    want = torch.zeros(n, dtype=torch.bool, device="cuda")
    want[(g.order[bad] // 3).long()] = True
    assert torch.equal(out, want[:, None].expand(n, d))


def test_no_picks():
    g = group_rows(torch.empty(5, 0, dtype=torch.int64, device="cuda"), 3)
    assert g.picks == 0 and g.n_rows == 5 and g.offsets.tolist() == [0] * 4
    X = torch.randn(5, 8, device="cuda")
    Y = rows_to_groups(X, g)
    assert Y.shape == (0, 8) and torch.equal(rows_from_groups(Y, g), torch.zeros_like(X))
    gY, gW = rows_from_groups_grad(X, Y, g, torch.empty(5, 0, device="cuda"))
    assert gY.shape == (0, 8) and gW.shape == (5, 0)


@pytest.mark.parametrize("n,k", [(100000, 100), (100000, 3000), (60000, 70000)])
def test_two_streams_at_once(n, k):
    """Sorts whose kernels overlap, on two streams at once and one behind the other."""
    jobs = []
    for s in range(2):
        lab = make_labels((n,), k, 50 + s, "skew")
        jobs.append((torch.cuda.Stream(), lab, group_rows(lab, k), []))
    torch.cuda.synchronize()
    for _ in range(8):
        for st, lab, _, got in jobs:
            with torch.cuda.stream(st):
                got.append(group_rows(lab, k))
    torch.cuda.synchronize()
    for _, _, want, got in jobs:
        for r in got:
            assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.parametrize("n", [1000, 4000])
def test_threads_with_sizes_of_their_own(n):
    """One kernel with little and with much shared memory, from two threads at once."""
    wrong = []

    def sort(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            lab = make_labels((n,), k, 60, "uniform")
            want = group_rows(lab, k)
            for _ in range(200):
                try:
                    got = group_rows(lab, k)
                except RuntimeError as e:
                    wrong.append(f"{k}: {e}")
                    return
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                wrong.append(f"{k}: other groups")

    threads = [threading.Thread(target=sort, args=(k,)) for k in (1500, 1900, 2040, 1700)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_groups_changed_before_the_backward_pass():
    g = group_rows(make_labels((20, 2), 4, 1), 4)
    X = torch.randn(20, 8, device="cuda", requires_grad=True)
    out = rows_from_groups(rows_to_groups(X, g), g)
    g.position.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_refusals():
    lab = make_labels((10, 2), 4, 1)
    g = group_rows(lab, 4)
    X = torch.randn(10, 8, device="cuda")
    with pytest.raises(RuntimeError, match="1D or 2D"):
        group_rows(lab.view(5, 2, 2), 4)
    with pytest.raises(RuntimeError, match="int64 or int32"):
        group_rows(lab.short(), 4)
    with pytest.raises(RuntimeError, match="contiguous"):
        group_rows(lab.t(), 4)
    with pytest.raises(RuntimeError, match="n_clusters"):
        group_rows(lab, -1)
    with pytest.raises(RuntimeError, match="10 rows"):
        rows_to_groups(X[:9], g)
    with pytest.raises(RuntimeError, match="contiguous"):
        rows_to_groups(X.t().contiguous().t(), g)
    Y = rows_to_groups(X, g)
    with pytest.raises(RuntimeError, match="20 rows"):
        rows_from_groups(X, g)
    with pytest.raises(RuntimeError, match="weights must be float32"):
        rows_from_groups(Y, g, torch.ones(10, 2, device="cuda").half())
    with pytest.raises(RuntimeError, match="weights must have shape"):
        rows_from_groups(Y, g, torch.ones(10, 3, device="cuda"))
    with pytest.raises(RuntimeError, match="grad_out must have shape"):
        rows_from_groups_grad(X[:, :4].contiguous(), Y, g)
    with pytest.raises(RuntimeError, match="fit together"):
        rows_to_groups(X, g._replace(order=g.order[:5]))
    with pytest.raises(RuntimeError, match="must be int32"):
        rows_to_groups(X, g._replace(order=g.order.long()))
    with pytest.raises(RuntimeError, match="X must be float32"):
        rows_to_groups(X.long(), g)


def test_positions_out_of_range_touch_nothing():
    """A RowGroups whose positions lie outside the slots: the kernels skip those slots."""
    g = group_rows(make_labels((10, 2), 4, 1), 4)
    pos = g.position.clone()
    pos[0, 0], pos[3, 1] = 20, 2 ** 31 - 1
    bad = g._replace(position=pos)
    X = torch.randn(10, 8, device="cuda")
    Y = torch.randn(20, 8, device="cuda")
    rows_to_groups(X, bad)
    W = torch.ones(10, 2, device="cuda")
    out = rows_from_groups(Y, bad, W)
    assert torch.equal(out[0], Y[int(g.position[0, 1])])
    gY, gW = rows_from_groups_grad(X, Y, bad, W)
    assert float(gW[0, 0]) == 0.0 and float(gW[3, 1]) == 0.0
