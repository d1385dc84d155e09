"""label_log_probs over scores that span their type: differences beyond it, whose log
probabilities are not, and the smallest and largest scales."""
import math

import numpy as np
import pytest
import torch

import label_reference as ref
from label_scores import label_log_probs, label_log_probs_grad

pytestmark = pytest.mark.gpu
WIDE = [torch.float32, torch.float64, torch.bfloat16]


def exact(x, scale):
    """(log p, p, entropy) of one row in 64 bits, its differences scaled before they are taken."""
    z = np.asarray([float(v) * 2.0 ** -10 for v in x.cpu().double()]) * scale  # exact but for the product
    hi = z.max()
    d = (z - hi) * 2.0 ** 10
    e = np.exp(d)
    log_p = d - math.log(e.sum())
    p = np.exp(log_p)
    return log_p, p, -np.where(p > 0, p * log_p, 0.0).sum()


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("m", [6, 300, 1001, 2048, 5000, 40001])
@pytest.mark.parametrize("factor", [0.25, -0.5])
def test_differences_beyond_the_type(dtype, m, factor):
    """Scores near both ends of the type: a difference of two is infinite, a log probability
    (scale times the difference) is not."""
    f = torch.finfo(dtype)
    x = torch.full((1, m), f.min / 2, device="cuda", dtype=dtype)
    x[0, m // 2], x[0, m // 2 + 1] = f.max * 0.75, f.max * 0.75
    x[0, 1], x[0, m - 1] = f.min, 0.0
    x = x * math.copysign(1, factor)
    for label in (0, 1, m // 2, m - 1):
        lab = torch.tensor([label], device="cuda")
        r = label_log_probs(x, lab, factor, 4)
        with np.errstate(all="ignore"):
            log_p, p, H = exact(x[0], factor)
        # the difference, its product and the logarithm: three roundings and that of log 2
        tol = 4 * ref.unit(dtype) * (np.abs(log_p) + 1)
        ref.close(r.log_probs, log_p[[label]], tol[[label]], "log_probs")
        ref.close(r.entropy, np.array([H]), np.array([8 * ref.unit(dtype)]), "entropy")
        ref.close(r.top_log_probs, log_p[r.top_labels.cpu().numpy()], tol[r.top_labels.cpu().numpy()], "top")
        assert r.top_labels[0, :3].tolist() == [m // 2, m // 2 + 1, m - 1]
        one = torch.ones(1, device="cuda", dtype=r.entropy.dtype)
        g = label_log_probs_grad(x, lab, r.row_stats, one, None, factor)
        want = factor * ((np.arange(m) == label) - p)
        ref.close(g, want[None], 8 * ref.unit(dtype) + ref.rounding(dtype, want[None]), "grad")


@pytest.mark.parametrize("dtype,least,most", [(torch.float32, -120, 126), (torch.bfloat16, -120, 126),
                                              (torch.float16, -126, 126), (torch.float64, -1014, 1022)])
@pytest.mark.parametrize("m", [5, 700, 9000])
def test_scales_at_their_limits(dtype, least, most, m):
    f = torch.finfo(dtype)
    x = torch.zeros(1, m, device="cuda", dtype=dtype)
    x[0, 1], x[0, 2] = f.max, f.min
    lab = torch.tensor([2], device="cuda")
    for scale in (2.0 ** least, -2.0 ** least):
        log_p, p, H = exact(x[0], scale)
        r = label_log_probs(x, lab, scale, 3)
        # log m and the sums' roundings: m / 128 + 24 additions
        tol = ref.unit(dtype) * (m / 128 + 40) * (np.abs(log_p) + math.log(m) + 1)
        ref.close(r.log_probs, log_p[[2]], tol[[2]], "log_probs")
        ref.close(r.entropy, np.array([H]), np.array([2 * tol.max()]), "entropy")
    r = label_log_probs(x, lab, 2.0 ** most, 1)
    assert int(r.top_labels) == 1 and float(r.entropy) == 0.0 and float(r.top_log_probs) == 0.0
    for scale in (2.0 ** (least - 1), -2.0 ** (least - 1)):
        with pytest.raises(RuntimeError, match="scale"):
            label_log_probs(x, lab, scale)
        with pytest.raises(RuntimeError, match="scale"):
            label_log_probs_grad(x, lab, r.row_stats, r.entropy, None, scale)
