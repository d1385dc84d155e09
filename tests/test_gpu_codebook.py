"""codebook.lookup and its gradient against the definitions, and the label operators run
together as the Lloyd loop's caller would."""
import numpy as np
import pytest
import torch

import label_reference as ref
from center_kernels import update_centers_fp32
from codebook import lookup, lookup_grad
from kmeans import LloydKMeans
from label_scores import label_log_probs
from row_groups import group_rows, rows_from_groups, rows_to_groups

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_labels(shape, k, seed, kind):
    g = gen(seed)
    if kind == "one":
        return torch.full(shape, k // 2, device="cuda", dtype=torch.int64)
    if kind == "none":
        return torch.full(shape, -1, device="cuda", dtype=torch.int64)
    if kind == "skew":
        u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
        return ((k + 1.0) ** u - 1).long().clamp_(0, k - 1)
    lab = torch.randint(0, k, shape, generator=g, device="cuda")
    if kind == "drop":
        r = torch.rand(shape, generator=g, device="cuda")
        lab = torch.where(r < 0.1, -5, torch.where(r > 0.8, k, lab))
    return lab


def check(C, G, lab, scale):
    k, d = C.shape
    dtype = C.dtype
    flat = lab.cpu().numpy().reshape(-1)
    ok = (flat >= 0) & (flat < k)
    s = float(torch.tensor(scale, dtype=torch.float64 if dtype == torch.float64 else torch.float32))
    want = np.where(ok[:, None], ref.f64(C)[np.where(ok, flat, 0)] * s, 0.0).reshape(*lab.shape, d)
    out = lookup(C, lab, scale)
    assert out.dtype == dtype and out.shape == (*lab.shape, d)
    u = ref.unit(dtype)
    ref.close(out, want, u * np.abs(want) + ref.rounding(dtype, want), "lookup")
    if scale == 1.0:
        assert np.array_equal(ref.f64(out), want)
    Gd = ref.f64(G).reshape(-1, d)
    total, size, count = np.zeros((k, d)), np.zeros((k, d)), np.zeros(k)
    np.add.at(total, flat[ok], Gd[ok] * s)
    np.add.at(size, flat[ok], np.abs(Gd[ok] * s))
    np.add.at(count, flat[ok], 1)
    tol = (count[:, None] + 2) * u * size + ref.rounding(dtype, total)
    got = lookup_grad(G, lab, k, scale)
    ref.close(got, total, tol, "lookup_grad")
    assert torch.equal(got, lookup_grad(G, lab, k, scale, groups=group_rows(lab.reshape(-1), k)))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["even", "drop", "one", "none", "skew"])
@pytest.mark.parametrize("n,k,d", [(1, 1, 1), (3, 5, 2048), (100, 7, 33), (1000, 50, 77), (5000, 300, 64),
                                   (700, 5000, 16), (2100, 1, 130), (90, 40, 515), (33, 9, 1001)])
def test_lookup_and_gradient(n, k, d, kind, dtype):
    g = gen(n + k + d)
    C = torch.randn(k, d, generator=g, device="cuda", dtype=torch.float64).to(dtype)
    G = torch.randn(n, d, generator=g, device="cuda", dtype=torch.float64).to(dtype)
    for scale in (1.0, -2.7):
        check(C, G, make_labels((n,), k, n, kind), scale)


@pytest.mark.parametrize("n,k,d,kind", [(300000, 100, 8, "even"), (200000, 3, 4, "skew"), (100000, 20, 24, "one"),
                                        (60000, 70000, 12, "skew")])
def test_long_labels(n, k, d, kind):
    """Labels with many rows, so that their sums cross many chunks."""
    g = gen(n)
    C = torch.randn(k, d, generator=g, device="cuda")
    G = torch.randn(n, d, generator=g, device="cuda")
    check(C, G, make_labels((n,), k, n, kind), 0.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k,d,kind", [(20000, 50, 45, "skew"), (3000, 1500, 333, "drop"), (1, 1, 33, "even"),
                                        (17, 2, 39, "one"), (4000, 3, 2049, "even"), (5000, 9000, 77, "skew"),
                                        (200000, 50, 45, "skew"), (30000, 1500, 333, "drop"), (160000, 2, 39, "one"),
                                        (100000, 90000, 77, "even"), (150000, 7, 33, "drop")])
def test_odd_rows_of_16_bits(n, k, d, kind, dtype):
    g = gen(n + d)
    C = torch.randn(k, d, generator=g, device="cuda", dtype=torch.float64).to(dtype)
    G = torch.randn(n, d, generator=g, device="cuda", dtype=torch.float64).to(dtype)
    lab = make_labels((n,), k, n, kind)
    got = check(C, G, lab, 0.75)
    # (neighbouring rows share 16-byte words: a NaN stays in its own label's row)
    G[n // 2] = float("nan")
    bad = lookup_grad(G, lab, k, 0.75).isnan()
    l = int(lab[n // 2])
    assert int(bad.sum()) == (d if 0 <= l < k else 0)
    assert not got.isnan().any() and (not 0 <= l < k or bad[l].all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_alignments_and_shapes(dtype, shift):
    g = gen(shift)

    def make(*s):
        n = int(np.prod(s))
        return torch.randn(n + shift, generator=g, device="cuda").to(dtype)[shift:].view(s)
    lab = make_labels((6, 35), 40, shift, "drop").to(torch.int32)
    check(make(40, 128), make(6, 35, 128), lab, 3.0)
    one = torch.tensor(7, device="cuda")  # a label of no dimension
    C = make(40, 128)
    assert torch.equal(lookup(C, one), C[7])


def test_empty():
    C = torch.randn(5, 8, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert lookup(C, none).shape == (0, 8)
    assert torch.equal(lookup_grad(torch.empty(0, 8, device="cuda"), none, 5), torch.zeros_like(C))
    assert lookup_grad(torch.empty(3, 0, device="cuda"), none.new_zeros(3), 5).shape == (5, 0)
    assert torch.equal(lookup(C[:0], none.new_zeros(3)), torch.zeros(3, 8, device="cuda"))
    assert lookup_grad(torch.ones(3, 8, device="cuda"), none.new_zeros(3), 0).shape == (0, 8)


def test_table_past_32_bit_elements():
    k, d = 270000, 8192  # 2.2e9 elements
    C = torch.empty(k, d, dtype=torch.float16, device="cuda")
    lab = torch.tensor([0, k - 1, k // 2, k - 1], device="cuda")
    rows = torch.randn(4, d, generator=gen(1), device="cuda").half()
    C[lab[:3]] = rows[:3]
    assert torch.equal(lookup(C, lab), C[lab])
    G = lookup_grad(rows, lab, k)
    assert torch.equal(G[0], rows[0]) and torch.equal(G[k // 2], rows[2])
    assert torch.equal(G[k - 1], (rows[1].float() + rows[3].float()).half()) and not G[k - 2].any()


def test_gradient_against_differences_and_autograd():
    lab = make_labels((4, 5), 6, 3, "drop")
    C = torch.randn(6, 3, generator=gen(1), device="cuda", dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda c: lookup(c, lab, 1.7), (C,))
    T = torch.randn(6, 40, device="cuda", requires_grad=True)
    lookup(T, lab, 2.0).sum().backward()  # a gradient of stride 0
    count = torch.stack([(lab == c).sum() for c in range(6)]).float()
    assert torch.equal(T.grad, (2.0 * count)[:, None].expand(6, 40))


def test_gradient_is_the_center_updates_sum():
    n, k, d = 20000, 50, 64
    X = torch.randn(n, d, generator=gen(1), device="cuda")
    lab = make_labels((n,), k, 2, "even")
    count = torch.bincount(lab, minlength=k).float()
    centers = update_centers_fp32(X, lab, k)
    got = lookup_grad(X, lab, k)
    mag = lookup_grad(X.abs(), lab, k)
    assert ((got / count[:, None] - centers).abs() <= (count[:, None] + 4) * 2.0 ** -23 * mag / count[:, None]).all()


def test_other_stream_captured_and_repeated():
    C = torch.randn(500, 96, generator=gen(1), device="cuda").bfloat16()
    lab = make_labels((9000,), 500, 4, "skew")

    def chain(lab):
        r = lookup(C, lab, 1.5)
        return r, lookup_grad(r, lab, 500, 0.5)
    want = chain(lab)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(lab)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    ls = torch.zeros_like(lab)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = chain(ls)
        graphs.append((g, got))
    ls.copy_(lab)
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    C = torch.randn(5, 8, device="cuda")
    lab = torch.zeros(4, dtype=torch.int64, device="cuda")
    G = torch.randn(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="C must be 2D"):
        lookup(C[0], lab)
    with pytest.raises(RuntimeError, match="C must be contiguous"):
        lookup(C.t(), lab)
    with pytest.raises(RuntimeError, match="int64 or int32"):
        lookup(C, lab.short())
    with pytest.raises(RuntimeError, match="C must be float32"):
        lookup(C.int(), lab)
    with pytest.raises(RuntimeError, match="labels' shape"):
        lookup_grad(G[:3], lab, 5)
    with pytest.raises(RuntimeError, match="belong"):
        lookup_grad(G, lab, 5, groups=group_rows(lab, 6))
    with pytest.raises(RuntimeError, match="belong"):
        lookup_grad(G, lab, 5, groups=group_rows(lab[:3], 5))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("op", ["fp16_fp32", "fp32_fp64", "double", "single", "tiled_bf16_fp32",
                                "tensorcore_fp16_fp64"])
def test_posterior(op):
    dt = torch.float64 if op == "double" else torch.float32
    C = torch.randn(40, 32, generator=gen(1), device="cuda", dtype=dt)
    X = C[torch.randint(0, 40, (777,), generator=gen(2), device="cuda")]
    X = (X + 0.5 * torch.randn(777, 32, generator=gen(3), device="cuda", dtype=dt)).contiguous()
    km = LloydKMeans(40, op=op, kappa=0.5)
    whole = km.posterior(X, C, temperature=3.0, top=4)
    labels = whole.top_labels[:, 1].contiguous()
    parts = km.posterior(X, C, temperature=3.0, labels=labels, top=4, block_rows=100)
    assert whole.log_probs is None
    for a, b in zip(whole[1:], parts[1:]):
        assert torch.equal(a, b)
    assert torch.equal(parts.log_probs, whole.top_log_probs[:, 1])
    # against the direct distances in 64 bits, within the distance operators' tolerance
    D = (X.double()[:, None] - C.double()[None]).square().sum(2)
    lp = torch.log_softmax(-D / 3.0, 1)
    tol = 8 * 2.0 ** -11 * (X.double().square().sum(1).max() + C.double().square().sum(1).max()) * 2 / 3.0
    tol = tol if op not in ("double", "single", "fp32_fp64") else tol * 2.0 ** -11
    assert float((whole.top_log_probs.double() - lp.gather(1, whole.top_labels)).abs().max()) <= float(tol)
    rows = km.reconstruct(C, parts.top_labels[:, 0].contiguous())
    assert torch.equal(rows, C[parts.top_labels[:, 0]])
    assert km.posterior(X[:0], C, top=2).top_labels.shape == (0, 2)


def test_soft_reconstruction_chain():
    """Points to their 3 likeliest centers, the residual of each taken there, and the weighted
    residuals brought back: forward and gradients against 64 bits."""
    n, k, d, p = 300, 20, 48, 3
    g = gen(11)
    C = torch.randn(k, d, generator=g, device="cuda", requires_grad=True)
    X = torch.randn(n, d, generator=g, device="cuda", requires_grad=True)
    R = torch.randn(n, d, generator=g, device="cuda")

    def loss(X, C):
        D = torch.cdist(X, C).square()
        r = label_log_probs(D, None, -0.5, p)
        lab = r.top_labels
        w = torch.log_softmax(-0.5 * D, 1).gather(1, lab).exp().contiguous()  # weights with a gradient
        groups = group_rows(lab, k)
        Y = rows_to_groups(X, groups) - lookup(C, groups.labels)
        out = rows_from_groups(Y, groups, w)
        return (out * R).sum() + r.entropy.sum(), lab

    def plain(X, C, lab):
        D = torch.cdist(X, C).square()
        lp = torch.log_softmax(-0.5 * D, 1)
        w = lp.gather(1, lab).exp()
        out = ((X[:, None] - C[lab]) * w[..., None]).sum(1)
        return (out * R.double()).sum() - (lp.exp() * lp).sum()
    got, lab = loss(X, C)
    gX, gC = torch.autograd.grad(got, (X, C))
    Xd, Cd = X.detach().double().requires_grad_(), C.detach().double().requires_grad_()
    want = plain(Xd, Cd, lab)
    wX, wC = torch.autograd.grad(want, (Xd, Cd))
    # D itself carries d * 2^-24 of |x|^2 + |c|^2 (about 100), which the exponent and its
    # gradient's factors (|x - c| of about 10) pass on
    tol = 48 * 2.0 ** -24 * 100 * 10
    assert abs(float((got - want).detach())) <= tol * n
    assert float((gX - wX).abs().max()) <= tol * float(wX.abs().max())
    assert float((gC - wC).abs().max()) <= tol * float(wC.abs().max())
