"""LloydKMeans.posterior refuses what it would answer wrongly; the refusals come before any
launch, so they need no GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from kmeans import LloydKMeans


def test_gradients_are_refused():
    x, c = torch.zeros(4, 3), torch.zeros(2, 3)
    km = LloydKMeans(2)
    for a, b in ((x.clone().requires_grad_(), c), (x, c.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="not differentiable"):
            km.posterior(a, b)
        with torch.no_grad(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            km.posterior(a, b)  # no gradient is recorded: the next check
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        km.posterior(x, fwAD.make_dual(c, torch.ones_like(c)))


def test_blocks_of_fewer_than_no_rows_are_refused():
    with pytest.raises(RuntimeError, match="block_rows"):
        LloydKMeans(2).posterior(torch.zeros(4, 3), torch.zeros(2, 3), block_rows=-5)


@pytest.mark.gpu
def test_without_recorded_gradients():
    g = torch.Generator(device="cuda").manual_seed(1)
    x, c = (torch.randn(n, 32, generator=g, device="cuda") for n in (50, 7))
    km = LloydKMeans(7)
    want = km.posterior(x, c, top=2)
    with torch.no_grad():
        got = km.posterior(x.requires_grad_(), c.requires_grad_(), top=2)
    assert all(torch.equal(a, b) for a, b in zip(want[1:], got[1:]))
    assert not got.entropy.requires_grad
