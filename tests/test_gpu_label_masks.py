"""label_log_probs over rows masked with a finite value (-1e4, the type's lowest), whose few
scores left lie side by side: the alternatives, exactly, and what they cost."""
import math

import pytest
import torch

from label_scores import label_log_probs
from test_gpu_label_scores import TYPES, check, gen

pytestmark = pytest.mark.gpu


def masked(n, m, dtype, kept, mask, seed, at=None):
    """Rows of `mask` but for `kept` neighbouring scores (beginning anywhere, or at `at`)."""
    g = gen(seed)
    x = torch.full((n, m), mask, device="cuda", dtype=dtype)
    for i in range(n):
        lo = int(torch.randint(0, m - kept + 1, (1,), generator=g, device="cuda")) if at is None else at
        x[i, lo:lo + kept] = torch.randn(kept, generator=g, device="cuda").to(dtype)
    return x


# fewer kept than the alternatives, a little more, more than a candidates' list holds
SHAPES = [(5, 60, 3, 8), (5, 64, 30, 8), (9, 250, 40, 8), (9, 250, 5, 30), (6, 251, 70, 6), (4, 500, 9, 16),
          (5, 509, 100, 16), (5, 1000, 50, 20), (5, 1024, 200, 32), (3, 1021, 4, 32), (700, 2000, 50, 5),
          (3, 2049, 20, 20), (1300, 3000, 40, 8), (3, 9001, 700, 32), (2, 32771, 7, 20), (2, 65537, 2000, 32),
          (1, 131072, 50, 20)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lowest", [True, False])
@pytest.mark.parametrize("n,m,kept,top", SHAPES)
def test_finite_masks(n, m, kept, top, lowest, dtype):
    mask = torch.finfo(dtype).min if lowest else -1e4
    x = masked(n, m, dtype, kept, mask, seed=m + kept)
    x[0, 0] = -math.inf  # a masked score of the other kind, which comes last
    lab = torch.arange(n, device="cuda") * 37 % m
    for rows in (slice(0, 4), slice(n - 2 if n > 2 else 0, n)):
        few, some = x[rows], lab[rows]
        check(few, some, 1.0, top, grads=False)
        check(-few, some, -1.0, top, grads=False)
    r, few = label_log_probs(x, lab, 1.0, top), label_log_probs(x[:4], lab[:4], 1.0, top)
    assert torch.equal(r.top_labels[:4], few.top_labels)  # among many rows as among few


@pytest.mark.parametrize("m,top", [(200, 8), (1000, 20), (2000, 8), (40000, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_finite_masks_and_equal_scores(m, top, dtype):
    """Half of a row at one value, half at another, with fewer scores above them than the
    alternatives; equal scores of both zeros; a tail of masks; +inf left of nothing else."""
    x = torch.full((6, m), -1e4, device="cuda", dtype=dtype)
    x[0, ::2] = -2e4
    x[0, m // 2:m // 2 + 3] = 1.0
    x[1, 1::2] = -2e4
    x[1, m - top + 1:] = torch.arange(top - 1, device="cuda").to(dtype)
    x[2, ::2], x[2, 1::2] = 0.0, -0.0
    x[2, 5] = 1.0
    x[3, : m // 2] = -math.inf
    x[4, : m - 2] = -math.inf  # fewer finite scores than alternatives
    x[5] = -math.inf
    x[5, ::3] = torch.finfo(dtype).min
    check(x, torch.tensor([0, 1, 2, m - 1, m - 1, 3], device="cuda"), 1.0, top, grads=False)
    y = torch.full((2, m), math.inf, device="cuda", dtype=dtype)  # +inf throughout: by index, NaN
    r = label_log_probs(y, None, 1.0, top)
    assert torch.equal(r.top_labels, torch.arange(top, device="cuda").expand(2, top))
    assert torch.isnan(r.top_log_probs).all() and torch.isnan(r.entropy).all()


def median_us(f, runs=7):
    f()
    times = []
    for _ in range(runs):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times)[runs // 2]


@pytest.mark.parametrize("n,m,dtype", [(4096, 131072, torch.bfloat16), (777, 32771, torch.float16),
                                       (16384, 8192, torch.float32), (65536, 3000, torch.bfloat16),
                                       (131072, 1024, torch.float32), (131072, 200, torch.float32)])
@pytest.mark.parametrize("kept,top", [(5, 8), (50, 20)])
def test_finite_masks_cost_what_other_rows_cost(n, m, dtype, kept, top):
    """At most six times the time of rows without a mask: the same single sweep, and a second
    look at the scores that reach the bound (by a search per alternative it is 9 to 195)."""
    x = torch.randn(n, m, generator=gen(m), device="cuda", dtype=torch.float32).to(dtype)
    plain = median_us(lambda: label_log_probs(x, None, 1.0, top))
    x[:, : m // 3] = -1e4
    x[:, m // 3 + kept:] = -1e4
    finite = median_us(lambda: label_log_probs(x, None, 1.0, top))
    assert finite <= 6 * plain, (finite, plain)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,top", [(40, 8), (250, 20), (500, 16), (1000, 20), (1021, 5), (2000, 8), (3000, 32), (9001, 4),
                                   (70001, 20)])
def test_rows_with_nan(m, top, dtype):
    """One NaN, a few, fewer than the alternatives or more, in one part of the row or throughout,
    among others, masked ones and equal ones: the NaN first, by index, then the others."""
    x = torch.randn(9, m, generator=gen(m), device="cuda").to(dtype)
    x[0, m // 2] = math.nan
    x[1, 1::2] = math.nan
    x[2, m - 3:] = math.nan
    x[3] = math.nan
    x[4] = -math.inf
    x[4, m // 3], x[4, 2] = math.nan, 1.0
    x[5] = 0.25
    x[5, m - 1] = math.nan
    x[6, 0], x[6, 1] = math.nan, math.inf
    x[7] = -1e4
    x[7, 3], x[7, m - 2] = math.nan, 0.5
    lab = torch.arange(9, device="cuda")
    check(x, lab, 1.0, top, grads=False)  # (row 8 has none)
    check(-x, lab, -1.0, top, grads=False)
    many = x.repeat(150, 1)
    r, few = label_log_probs(many, None, 1.0, top), label_log_probs(x, None, 1.0, top)
    assert torch.equal(r.top_labels, few.top_labels.repeat(150, 1))


@pytest.mark.parametrize("n,m,dtype", [(4096, 131072, torch.bfloat16), (65536, 3000, torch.bfloat16)])
def test_rows_of_nan_cost_what_other_rows_cost(n, m, dtype):
    """A training step that has gone wrong: nothing but NaN (six times as above)."""
    x = torch.randn(n, m, generator=gen(m), device="cuda", dtype=torch.float32).to(dtype)
    plain = median_us(lambda: label_log_probs(x, None, 1.0, 20))
    x.fill_(math.nan)
    assert median_us(lambda: label_log_probs(x, None, 1.0, 20)) <= 6 * plain
