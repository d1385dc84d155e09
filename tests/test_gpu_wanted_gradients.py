"""The autograd forms keep and form what the wanted gradients need, and no more."""
import pytest
import torch

import label_scores
from row_groups import group_rows, rows_from_groups, rows_from_groups_grad

pytestmark = pytest.mark.gpu
N, P, K, D = 4000, 3, 7, 512


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.fixture
def grouped():
    lab = torch.randint(-1, K + 1, (N, P), generator=gen(1), device="cuda")  # some are dropped
    groups = group_rows(lab, K)
    Y = torch.randn(N * P, D, generator=gen(2), device="cuda")
    W = torch.rand(N, P, generator=gen(3), device="cuda")
    G = torch.randn(N, D, generator=gen(4), device="cuda")
    return groups, Y, W, G


def test_rows_back_without_weights_keep_no_rows(grouped):
    groups, Y, _, G = grouped
    leaf = Y.clone().requires_grad_()
    Z = leaf * 1.0
    out = rows_from_groups(Z, groups)
    Z.mul_(2.0)  # Y is not needed again
    out.backward(G)
    assert torch.equal(leaf.grad, rows_from_groups_grad(G, Y, groups)[0])


def test_rows_back_with_frozen_weights_keep_no_rows(grouped):
    groups, Y, W, G = grouped
    leaf = Y.clone().requires_grad_()
    Z = leaf * 1.0
    out = rows_from_groups(Z, groups, W)
    Z.zero_()
    out.backward(G)
    assert torch.equal(leaf.grad, rows_from_groups_grad(G, Y, groups, W)[0])
    assert W.grad is None


def test_rows_back_with_frozen_rows_form_no_row_gradient(grouped):
    groups, Y, W, G = grouped
    want = rows_from_groups_grad(G, Y, groups, W)[1]
    leaf = W.clone().requires_grad_()
    weights = leaf * 1.0
    out = rows_from_groups(Y, groups, weights)
    weights.zero_()  # the weights are needed for the rows' gradient alone
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out.backward(G)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < Y.numel() * 4 // 2
    assert torch.equal(leaf.grad, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,p,d", [(1, 1, 1), (5, 2, 7), (17, 3, 33), (64, 8, 256), (100, 5, 1001), (9, 1, 4100),
                                   (5, 3, 0), (0, 2, 8)])
def test_one_gradient_at_a_time(n, p, d, dtype):
    """As both together, bit by bit."""
    groups = group_rows(torch.randint(-1, 5, (n, p), generator=gen(n + d), device="cuda"), 4)
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    Y = torch.randn(n * p, d, generator=gen(5), device="cuda", dtype=acc).to(dtype)
    G = torch.randn(n, d, generator=gen(6), device="cuda", dtype=acc).to(dtype)
    W = torch.randn(n, p, generator=gen(7), device="cuda", dtype=acc)
    want = rows_from_groups_grad(G, Y, groups, W)
    a, b = Y.clone().requires_grad_(), W.clone().requires_grad_()
    rows_from_groups(a, groups, W).backward(G)
    rows_from_groups(Y, groups, b).backward(G)
    assert torch.equal(a.grad, want[0]) and torch.equal(b.grad, want[1])
    a.grad = b.grad = None
    rows_from_groups(a, groups, b).backward(G)
    assert torch.equal(a.grad, want[0]) and torch.equal(b.grad, want[1])


def test_outputs_outside_the_loss_cost_nothing(monkeypatch):
    """A loss through one output alone: no gradient of zeros for the other is made or read."""
    seen = []
    real = label_scores.label_log_probs_grad

    def spy(scores, labels, stats, grad_log_probs=None, grad_entropy=None, scale=1.0):
        seen.append((grad_log_probs is not None, grad_entropy is not None))
        return real(scores, labels, stats, grad_log_probs, grad_entropy, scale)
    monkeypatch.setattr(label_scores, "label_log_probs_grad", spy)
    x = torch.randn(50, 333, generator=gen(1), device="cuda").requires_grad_()
    lab = torch.arange(50, device="cuda")
    one = torch.ones(50, device="cuda")
    for labels, pick, want in ((lab, lambda r: r.log_probs, (True, False)), (lab, lambda r: r.entropy, (False, True)),
                               (None, lambda r: r.entropy, (False, True)),
                               (lab, lambda r: r.log_probs + r.entropy, (True, True))):
        x.grad = None
        r = label_scores.label_log_probs(x, labels, 1.5, 2)
        pick(r).sum().backward()
        assert seen.pop() == want and not seen
        assert torch.equal(x.grad, real(x.detach(), labels, r.row_stats, one if want[0] else None,
                                        one if want[1] else None, 1.5))
