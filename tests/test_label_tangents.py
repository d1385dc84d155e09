"""The label operators refuse inputs with forward-mode tangents, whose derivative they would
drop; the refusal comes before any other check, so it needs no GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import codebook
import label_scores
import row_groups

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_tangents_are_refused(device):
    x, w = torch.ones(4, 3, device=device), torch.ones(4, 2, device=device)
    lab = torch.zeros(4, dtype=torch.int64, device=device)
    slots = torch.zeros(8, dtype=torch.int32, device=device)
    groups = row_groups.RowGroups(torch.zeros(4, dtype=torch.int32, device=device), slots, slots.view(4, 2), slots)
    y, one, stats = torch.ones(8, 3, device=device), torch.ones(4, device=device), torch.ones(4, 3, device=device)
    calls = (lambda d: label_scores.label_log_probs(d(x), lab),
             lambda d: label_scores.label_log_probs_grad(d(x), lab, stats, one),
             lambda d: row_groups.rows_to_groups(d(x), groups),
             lambda d: row_groups.rows_from_groups(d(y), groups),
             lambda d: row_groups.rows_from_groups(y, groups, d(w)),
             lambda d: codebook.lookup(d(x), lab),
             lambda d: codebook.lookup_grad(d(x), lab, 3))
    if device == "cuda":  # (these look at the other arguments first)
        calls += (lambda d: label_scores.label_log_probs(d(x).requires_grad_(), lab),
                  lambda d: label_scores.label_log_probs_grad(x, lab, stats, d(one)),
                  lambda d: label_scores.label_log_probs_grad(x, lab, stats, None, d(one)),
                  lambda d: row_groups.rows_from_groups_grad(d(x), y, groups, w),
                  lambda d: row_groups.rows_from_groups_grad(x, d(y), groups, w),
                  lambda d: row_groups.rows_from_groups_grad(x, y, groups, d(w)))
    with fwAD.dual_level():
        for f in calls:
            with pytest.raises((RuntimeError, NotImplementedError), match="forward-mode|jvp"):
                f(lambda t: fwAD.make_dual(t.clone(), torch.ones_like(t)))
        if device == "cuda":  # without a tangent, an open level changes nothing
            assert label_scores.label_log_probs(x, lab).entropy.shape == (4,)
            assert codebook.lookup(x, lab).shape == (4, 3)
