"""label_log_probs and its gradient against the definitions in 64 bits: types, sizes from one
column to many, strides, masks, ties, infinities and NaN, streams and captured graphs."""
import math

import numpy as np
import pytest
import torch

import label_reference as ref
from _lib import call_on, lib
from label_scores import label_log_probs, label_log_probs_grad

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(n, m, dtype, seed, pad=0, spread=3.0, offset=0.0):
    g = gen(seed)
    buf = (torch.randn(n, m + pad, generator=g, device="cuda", dtype=torch.float64) * spread + offset).to(dtype)
    lab = torch.randint(0, m, (n,), generator=g, device="cuda")
    return buf[:, :m], lab


def check(x, lab, scale=1.0, top=0, grads=True):
    n, m = x.shape
    r = label_log_probs(x, lab, scale, top)
    lp, H, tlp, tl, p, log_p = ref.label_scores(x, lab, scale, top)
    tL, tH, tp = ref.score_bounds(m, x.dtype, log_p)
    ref.close(r.entropy, H, tH, "entropy")
    if lab is not None:
        ok = ((lab >= 0) & (lab < m)).cpu().numpy()
        at = np.where(ok, lab.cpu().numpy(), 0)
        ref.close(r.log_probs, lp, tp[np.arange(n), at], "log_probs")
    else:
        assert r.log_probs is None
    assert np.array_equal(r.top_labels.cpu().numpy(), tl)
    ref.close(r.top_log_probs, tlp, np.take_along_axis(tp, tl, 1), "top_log_probs")
    if grads:
        g = gen(n * 7 + m)
        acc = r.entropy.dtype
        gl = torch.randn(n, generator=g, device="cuda", dtype=acc)
        ge = torch.randn(n, generator=g, device="cuda", dtype=acc)
        for a, b in ((gl, ge), (gl, None), (None, ge)):
            if lab is None and a is not None:
                continue
            want, tol = ref.label_scores_grad(p, log_p, H, lab, scale, a, b, x.dtype)
            got = label_log_probs_grad(x, lab, r.row_stats, a, b, scale)
            assert got.dtype == x.dtype and got.is_contiguous()
            ref.close(got, want, tol, "grad")
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m,top", [(1, 1, 1), (3, 2, 2), (5, 7, 7), (33, 31, 8), (4, 32, 32), (17, 33, 5),
                                     (9, 257, 32), (130, 1000, 8), (65, 1024, 1), (3, 2049, 20), (2, 4096, 32),
                                     (7, 9973, 32), (2, 65537, 20), (1, 131072, 32)])
def test_sizes(dtype, n, m, top):
    x, lab = make(n, m, dtype, seed=n + m)
    check(x, lab, 1.0, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.5, 2.5, 1e-3, -30.0])
@pytest.mark.parametrize("n,m,pad", [(19, 515, 3), (6, 4100, 13), (40, 64, 1)])
def test_scales_and_row_strides(dtype, scale, n, m, pad):
    x, lab = make(n, m, dtype, seed=m, pad=pad)
    check(x, lab.to(torch.int32), scale, 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_alignments(dtype, shift):
    n, m = 5, 1031
    flat = torch.randn(shift + n * m, generator=gen(3), device="cuda").to(dtype)
    x = flat[shift:shift + n * m].view(n, m)
    check(x, torch.arange(n, device="cuda"), 1.0, 6)


@pytest.mark.parametrize("m,top", [(1, 1), (40, 32), (1500, 8), (20000, 20), (140000, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_scores_go_by_index(dtype, m, top):
    x = torch.full((3, m), 0.25, device="cuda", dtype=dtype)
    x[1, m // 2:] = 0.5
    x[2] = torch.randint(0, 3, (m,), generator=gen(m), device="cuda").to(dtype)
    check(x, torch.tensor([0, m - 1, m // 2], device="cuda"), 1.0, top)
    check(x, torch.tensor([0, m - 1, m // 2], device="cuda"), -2.0, top)


@pytest.mark.parametrize("n,m,top", [(5, 60, 8), (5, 250, 30), (3, 1000, 20), (3, 2000, 8), (700, 2000, 5),
                                     (2, 9000, 32), (1300, 3000, 8), (1300, 9001, 4), (2, 100003, 32), (1, 131072, 20)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_sorted_and_stepped_rows(n, m, top, dtype):
    """Rows whose best scores lie together: rising, falling, in steps of equal ones, and nearly
    all equal; far more scores than the candidates' list holds reach any early bound."""
    ramp = torch.arange(m, device="cuda", dtype=torch.float32)
    rows = [ramp / m, -ramp / m, (ramp / 700).floor(), -(ramp / 700).floor(), torch.zeros_like(ramp),
            (ramp % 2), torch.where(ramp == m // 2, 1.0, 0.0)]
    x = torch.stack([rows[i % len(rows)] for i in range(n)]).to(dtype)
    lab = torch.arange(n, device="cuda") % m
    check(x[:7], lab[:7], 1.0, top, grads=False)
    r, few = label_log_probs(x, lab, 1.0, top), label_log_probs(x[:7], lab[:7], 1.0, top)
    for i in range(0, n, 97):  # a row among many as a row among few, whichever kernel takes it
        if i % 7 < min(7, n):
            assert torch.equal(r.top_labels[i], few.top_labels[i % 7])


def test_zeros_of_both_signs_are_equal():
    x = torch.zeros(2, 100, device="cuda")
    x[0, ::2] = -0.0
    x[1, 1::2] = -0.0
    check(x, torch.tensor([3, 4], device="cuda"), 1.0, 10)
    check(x, torch.tensor([3, 4], device="cuda"), -1.0, 10)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,left", [(37, 0), (37, 1), (37, 3), (600, 1), (5000, 2), (70000, 3), (70000, 40000)])
@pytest.mark.parametrize("scale", [1.0, -0.7])
def test_masked(dtype, m, left, scale):
    """Rows with `left` scores kept (none, fewer than the alternatives, many); the others are
    -inf in z.  Masked labels have log probability -inf."""
    n = 6
    x, lab = make(n, m, dtype, seed=left + m)
    x = x.clone()
    for i in range(n):
        drop = torch.randperm(m, generator=gen(i), device="cuda")[left:]
        x[i, drop] = -math.inf * math.copysign(1, scale)
    lab[0] = int(torch.isinf(x[0]).nonzero()[0])
    check(x, lab, scale, min(m, 9))


@pytest.mark.parametrize("dtype", TYPES)
def test_lowest_value_as_mask(dtype):
    """A mask of the type's lowest value is a finite score: a row of nothing else is uniform."""
    lo = torch.finfo(dtype).min
    for m in (50, 3000):
        x, lab = make(5, m, dtype, seed=m)
        x = x.clone()
        x[0, ::2] = lo
        x[1] = lo
        x[2, : m - 1] = lo
        x[3] = -lo
        x[4, 1:] = lo
        x[4, 0] = torch.finfo(dtype).max / 2
        lab[4] = 0
        check(x[:4], lab[:4], 1.0, 4)
        r = label_log_probs(x[4:], lab[4:], 1.0, 2)  # lowest - largest may overflow: probability 0
        assert float(r.log_probs[0]) == 0.0 and float(r.entropy[0]) == 0.0
        g = label_log_probs_grad(x[4:], lab[4:], r.row_stats, torch.ones(1, device="cuda", dtype=r.entropy.dtype),
                                 torch.ones(1, device="cuda", dtype=r.entropy.dtype))
        assert torch.equal(g, torch.zeros_like(g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [20, 900, 40000])
def test_nan_and_infinity(dtype, m):
    x, lab = make(5, m, dtype, seed=m)
    x = x.clone()
    x[0, m // 3] = math.nan
    x[1, m - 1] = math.inf
    x[2, 0], x[2, 5] = math.nan, math.inf
    x[3, 1::2] = math.nan
    r = check(x, lab, 1.0, 6, grads=False)
    assert torch.isnan(r.log_probs[:4]).all() and torch.isnan(r.entropy[:4]).all()
    g = label_log_probs_grad(x, lab, r.row_stats, torch.ones_like(r.entropy), torch.ones_like(r.entropy))
    assert torch.isnan(g[:4]).all() and torch.isfinite(g[4]).all()
    check(x, lab, -1.0, 6, grads=False)  # +inf is a masked score there


@pytest.mark.parametrize("m", [3, 700, 30000])
def test_common_offset_and_far_tails(m):
    """Scores near 1e6 with differences of order one, and rows that span hundreds."""
    x, lab = make(7, m, torch.float32, seed=m, spread=2.0, offset=1e6)
    check(x, lab, -1.0, 3)
    y, lab = make(7, m, torch.float32, seed=m, spread=200.0)
    check(y, lab, 1.0, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_labels_outside_and_none(dtype):
    x, lab = make(8, 77, dtype, seed=1)
    lab[0], lab[3], lab[5] = -1, 77, 2 ** 40
    r = check(x, lab, 1.0, 2)
    assert (r.log_probs[[0, 3, 5]] == 0).all()
    check(x, None, 1.0, 2)
    assert label_log_probs(x[:0], lab[:0], 1.0, 2).top_labels.shape == (0, 2)


@pytest.mark.parametrize("dtype", [torch.float16])
def test_rows_past_32_bit_offsets(dtype):
    """Row starts beyond 2^31 elements (a wide buffer of which few columns are read)."""
    n, m, ld = 3, 2000, (1 << 30) + 8
    buf = torch.empty(2 * ld + m, dtype=dtype, device="cuda")
    x = buf.as_strided((n, m), (ld, 1))
    for i in range(n):
        x[i] = torch.randn(m, generator=gen(i), device="cuda").to(dtype)
    check(x, torch.arange(n, device="cuda"), 1.0, 4)


def test_many_rows_past_32_bit_elements():
    n, m = 70000, 32768  # 2.3e9 elements; first, middle and last rows against the reference
    x = torch.empty(n, m, dtype=torch.bfloat16, device="cuda")
    for lo in range(0, n, 10000):
        x[lo:lo + 10000] = torch.randn(min(10000, n - lo), m, generator=gen(lo), device="cuda").to(x.dtype)
    lab = torch.arange(n, device="cuda") % m
    r = label_log_probs(x, lab, 1.0, 3)
    ge = torch.ones(n, device="cuda")
    g = label_log_probs_grad(x, lab, r.row_stats, ge, ge)
    for lo in (0, 34999, n - 5):
        rows = slice(lo, lo + 5)
        lp, H, tlp, tl, p, log_p = ref.label_scores(x[rows], lab[rows], 1.0, 3)
        tL, tH, tp = ref.score_bounds(m, x.dtype, log_p)
        ref.close(r.log_probs[rows], lp, tp[np.arange(5), lab[rows].cpu().numpy()], "log_probs")
        ref.close(r.entropy[rows], H, tH, "entropy")
        assert np.array_equal(r.top_labels[rows].cpu().numpy(), tl)
        want, tol = ref.label_scores_grad(p, log_p, H, lab[rows], 1.0, ge[:5], ge[:5], x.dtype)
        ref.close(g[rows], want, tol, "grad")


@pytest.mark.parametrize("m", [6, 300])
def test_gradient_against_differences(m):
    x, lab = make(3, m, torch.float64, seed=m)
    lab[1] = -1
    x = x.clone().requires_grad_()

    def f(t):
        r = label_log_probs(t, lab, -0.8, 2)
        return r.log_probs, r.entropy
    assert torch.autograd.gradcheck(f, (x,), eps=1e-6, atol=1e-6, rtol=1e-5)


def test_autograd_in_the_scores_type_and_broadcast_gradients():
    x, lab = make(5, 333, torch.bfloat16, seed=2)
    x = x.clone().requires_grad_()
    r = label_log_probs(x, lab, 1.5, 3)
    assert not r.top_log_probs.requires_grad and not r.row_stats.requires_grad
    (r.log_probs.sum() + 0.1 * r.entropy.sum()).backward()  # expanded (stride 0) gradients
    one = torch.ones(5, device="cuda")
    want = label_log_probs_grad(x.detach(), lab, r.row_stats, one, 0.1 * one, 1.5)
    assert torch.equal(x.grad, want)
    x.grad = None
    label_log_probs(x, lab, 1.5).entropy.sum().backward()
    assert torch.equal(x.grad, label_log_probs_grad(x.detach(), lab, r.row_stats, None, one, 1.5))


def test_autograd_without_labels_or_rows():
    x, _ = make(4, 50, torch.float32, seed=6)
    x = x.clone().requires_grad_()
    r = label_log_probs(x, None, 0.5, 2)
    assert r.log_probs is None
    r.entropy.sum().backward()
    one = torch.ones(4, device="cuda")
    assert torch.equal(x.grad, label_log_probs_grad(x.detach(), None, r.row_stats, None, one, 0.5))
    e = torch.empty(0, 50, device="cuda", requires_grad=True)
    label_log_probs(e, torch.empty(0, dtype=torch.int64, device="cuda")).log_probs.sum().backward()
    assert e.grad.shape == (0, 50)


def test_two_streams_at_once():
    """The same calls on two streams, interleaved, with inputs of their own."""
    jobs = []
    for s in range(2):
        x, lab = make(300, 20000, torch.bfloat16, seed=40 + s)
        jobs.append((torch.cuda.Stream(), x, lab, label_log_probs(x, lab, 1.0, 8), []))
    torch.cuda.synchronize()
    for _ in range(6):
        for st, x, lab, _, got in jobs:
            with torch.cuda.stream(st):
                got.append(label_log_probs(x, lab, 1.0, 8))
    torch.cuda.synchronize()
    for _, _, _, want, got in jobs:
        for r in got:
            assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.parametrize("n,m", [(1, 131072), (300, 1000), (3, 40000)])
def test_same_result_every_time_and_any_place(n, m):
    """A row's outputs do not depend on the run, nor on the other rows."""
    x, lab = make(n, m, torch.float32, seed=5)
    a, b = label_log_probs(x, lab, 1.0, 8), label_log_probs(x, lab, 1.0, 8)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_other_stream_and_captured():
    x, lab = make(4, 50000, torch.bfloat16, seed=9)
    want = label_log_probs(x, lab, 1.0, 6)
    one = torch.ones(4, device="cuda")
    want_g = label_log_probs_grad(x, lab, want.row_stats, one, one)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = label_log_probs(x, lab, 1.0, 6)
        got_g = label_log_probs_grad(x, lab, got.row_stats, one, one)
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want)) and torch.equal(got_g, want_g)
    xs = torch.zeros_like(x)
    graphs = []
    for _ in range(2):  # two graphs over the same inputs
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = label_log_probs(xs, lab, 1.0, 6)
            d = label_log_probs_grad(xs, lab, r.row_stats, one, one)
        graphs.append((g, r, d))
    xs.copy_(x)
    for g, r, d in graphs:
        g.replay()
    torch.cuda.synchronize()
    for g, r, d in graphs:
        assert all(torch.equal(u, v) for u, v in zip(r, want)) and torch.equal(d, want_g)


def test_refusals():
    x, lab = make(4, 9, torch.float32, seed=1)
    for bad, what in ((dict(top=10), "top"), (dict(top=-1), "top"), (dict(scale=0.0), "scale"),
                      (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale")):
        with pytest.raises(RuntimeError, match=what):
            label_log_probs(x, lab, **bad)
    with pytest.raises(RuntimeError, match="top"):
        label_log_probs(torch.zeros(1, 100, device="cuda"), None, top=33)
    with pytest.raises(RuntimeError, match="contiguous"):
        label_log_probs(torch.zeros(9, 4, device="cuda").t(), None)
    with pytest.raises(RuntimeError, match="overlap"):
        label_log_probs(torch.zeros(1, 9, device="cuda").expand(4, 9), lab)
    with pytest.raises(RuntimeError, match="shape"):
        label_log_probs(x, lab[:3])
    with pytest.raises(RuntimeError, match="int64 or int32"):
        label_log_probs(x, lab.float())
    with pytest.raises(RuntimeError, match="scores must be float32"):
        label_log_probs(x.long(), lab)
    with pytest.raises(RuntimeError, match="2D"):
        label_log_probs(x[0], lab)
    with pytest.raises(RuntimeError, match="column"):
        label_log_probs(x[:, :0], lab)
    r = label_log_probs(x, lab)
    with pytest.raises(RuntimeError, match="needs labels"):
        label_log_probs_grad(x, None, r.row_stats, r.entropy)
    with pytest.raises(RuntimeError, match="row_stats"):
        label_log_probs_grad(x, lab, r.row_stats[:3], r.entropy)
    with pytest.raises(RuntimeError, match="grad_entropy must be float32"):
        label_log_probs_grad(x, lab, r.row_stats, None, r.entropy.double())
    with pytest.raises(RuntimeError, match="null pointer"):
        call_on(x, lib().euc_label_log_probs, 0, x.data_ptr(), 9, 4, 9, None, 1, 1.0, 0, r.entropy.data_ptr(), None,
                None, None, None)
