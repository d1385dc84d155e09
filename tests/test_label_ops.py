"""Host side of the label operators (no GPU): public names and defaults, refusals, and the
C ABI's checks, which come before the device's."""
import ctypes
import inspect
import os

import pytest
import torch

import codebook
import kmeans
import label_scores
import row_groups

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E = inspect.Parameter.empty


def sig(f):
    return [(p.name, p.default) for p in inspect.signature(f).parameters.values()]


def test_names_and_defaults():
    assert sig(label_scores.label_log_probs) == [("scores", E), ("labels", None), ("scale", 1.0), ("top", 0)]
    assert sig(label_scores.label_log_probs_grad) == [("scores", E), ("labels", E), ("row_stats", E),
                                                      ("grad_log_probs", None), ("grad_entropy", None),
                                                      ("scale", 1.0)]
    assert sig(row_groups.group_rows) == [("labels", E), ("n_clusters", E)]
    assert sig(row_groups.rows_to_groups) == [("X", E), ("groups", E)]
    assert sig(row_groups.rows_from_groups) == [("Y", E), ("groups", E), ("weights", None)]
    assert sig(row_groups.rows_from_groups_grad) == [("grad_out", E), ("Y", E), ("groups", E), ("weights", None)]
    assert sig(codebook.lookup) == [("C", E), ("labels", E), ("scale", 1.0)]
    assert sig(codebook.lookup_grad) == [("G", E), ("labels", E), ("n_clusters", E), ("scale", 1.0),
                                         ("groups", None)]
    for f in ("posterior", "reconstruct"):
        assert hasattr(kmeans.LloydKMeans, f)


def test_cpu_tensors_are_refused():
    x, lab = torch.zeros(4, 3), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="scores must be a CUDA tensor"):
        label_scores.label_log_probs(x, lab)
    with pytest.raises(RuntimeError, match="labels must be a CUDA tensor"):
        row_groups.group_rows(lab, 3)
    with pytest.raises(RuntimeError, match="C must be a CUDA tensor"):
        codebook.lookup(x, lab)
    with pytest.raises(RuntimeError, match="G must be a CUDA tensor"):
        codebook.lookup_grad(x, lab, 3)
    with pytest.raises(TypeError):
        label_scores.label_log_probs(x.numpy(), lab)
    with pytest.raises(TypeError, match="RowGroups"):
        row_groups.rows_to_groups(x, (lab,))
    with pytest.raises(RuntimeError, match="temperature"):
        kmeans.LloydKMeans(3).posterior(x, x, temperature=0.0)
    with pytest.raises(RuntimeError, match="labels must have shape"):
        kmeans.LloydKMeans(3).posterior(x, x, labels=torch.zeros(5, dtype=torch.int64))


@pytest.fixture(scope="module")
def lib():
    import _lib
    return _lib.lib()


NO_GPU = not torch.cuda.is_available()
P = ctypes.c_void_p(256)


def test_scores_abi_checks(lib):
    f = lib.euc_label_log_probs

    def call(t=0, x=P, ld=8, n=4, m=8, lab=P, scale=1.0, top=0, lp=None, tlp=None, tl=None):
        return f(t, x, ld, n, m, lab, 1, scale, top, lp, None, None, tlp, tl, None)
    assert call(t=4) == 2 and call(t=-1) == 2                       # EUC_ERR_DTYPE
    assert call(n=-1) == 1 and call(m=0) == 1 and call(ld=7) == 1   # EUC_ERR_SHAPE
    assert call(m=2 ** 31 - 1, ld=2 ** 31) == 1
    assert call(scale=0.0) == 7 and call(scale=float("nan")) == 7 and call(scale=float("inf")) == 7
    assert call(top=9) == 3 and call(top=-1) == 3 and call(m=64, ld=64, top=33) == 3
    if NO_GPU:
        assert call() == 8
    else:  # refused before any launch
        assert call(x=None) == 7 and call(lab=None, lp=P) == 7 and call(top=1) == 7
        assert call(x=ctypes.c_void_p(258)) == 7 and call(n=0) == 0
        off4, off2 = ctypes.c_void_p(260), ctypes.c_void_p(258)
        assert call(lab=off4, lp=P) == 7 and call(lp=off2) == 7 and call(top=1, tlp=P, tl=off4) == 7
    g = lib.euc_label_log_probs_grad
    assert g(0, P, 8, 4, 8, P, 1, 0.0, P, P, None, P, None) == 7
    assert g(0, P, 7, 4, 8, P, 1, 1.0, P, P, None, P, None) == 1
    if not NO_GPU:
        assert g(0, P, 8, 4, 8, None, 1, 1.0, P, P, None, P, None) == 7
        assert g(0, P, 8, 4, 8, P, 1, 1.0, None, P, None, P, None) == 7
        assert g(0, P, 8, 4, 8, P, 1, 1.0, off2, P, None, P, None) == 7
        assert g(1, P, 8, 4, 8, P, 1, 1.0, P, off4, None, P, None) == 7


def test_groups_abi_checks(lib):
    big = 2 ** 31 - 1
    assert lib.euc_group_rows_workspace_bytes(0, 5) == 0
    assert lib.euc_group_rows_workspace_bytes(big, 5) == 0 and lib.euc_group_rows_workspace_bytes(5, big) == 0
    # one block, one pass: none; several passes keep keys and slots between them; many slots
    # keep a histogram per tile too
    assert lib.euc_group_rows_workspace_bytes(1000, 64) == 0
    assert lib.euc_group_rows_workspace_bytes(1000, 100000) >= 2 * 4000
    assert lib.euc_group_rows_workspace_bytes(1 << 20, 64) >= 65 * 256 * 4
    f = lib.euc_group_rows
    assert f(P, 1, -1, 4, P, P, P, P, P, 1 << 20, None) == 1 and f(P, 1, 4, -1, P, P, P, P, P, 1 << 20, None) == 1
    assert f(P, 1, big, 4, P, P, P, P, P, 1 << 20, None) == 1 and f(P, 1, 4, big, P, P, P, P, P, 1 << 20, None) == 1
    t, b, g = lib.euc_rows_to_groups, lib.euc_rows_from_groups, lib.euc_rows_from_groups_grad
    assert t(9, P, P, P, 4, 2, 8, P, None) == 2 and t(0, P, P, P, -4, 2, 8, P, None) == 1
    assert t(0, P, P, P, 1 << 20, 1 << 12, 8, P, None) == 1
    assert b(0, P, P, P, 4, 2, -8, P, None) == 1 and g(0, P, P, P, P, P, 4, -2, 8, P, P, None) == 1
    if NO_GPU:
        assert f(P, 1, 4, 4, P, P, P, P, P, 1 << 20, None) == 8 and t(0, P, P, P, 4, 2, 8, P, None) == 8
        assert b(0, P, P, P, 4, 2, 8, P, None) == 8 and g(0, P, P, P, P, P, 4, 2, 8, P, P, None) == 8
    else:
        assert f(P, 1, 4, 10000, P, P, P, P, P, 16, None) == 6      # EUC_ERR_WORKSPACE
        assert f(P, 1, 4, 10000, P, P, P, P, ctypes.c_void_p(264), 1 << 20, None) == 7  # workspace off 16 bytes
        assert f(P, 1, 4, 4, P, None, P, P, P, 1 << 20, None) == 7
        assert t(0, None, P, P, 4, 2, 8, P, None) == 7 and b(0, P, P, P, 4, 2, 8, None, None) == 7
        assert t(0, ctypes.c_void_p(258), P, P, 4, 2, 8, P, None) == 7
        assert g(0, P, None, P, P, P, 4, 2, 8, P, P, None) == 7
        off = ctypes.c_void_p(258)
        assert f(P, 1, 4, 4, P, off, P, P, P, 1 << 20, None) == 7 and f(off, 0, 4, 4, P, P, P, P, P, 0, None) == 7
        assert t(2, P, off, P, 4, 2, 8, P, None) == 7 and b(2, P, P, off, 4, 2, 8, P, None) == 7
        assert g(2, P, P, P, P, P, 4, 2, 8, P, off, None) == 7


def test_codebook_abi_checks(lib):
    f, g = lib.euc_codebook_lookup, lib.euc_codebook_grad
    assert f(7, P, 4, P, 1, 4, 8, 1.0, P, None) == 2
    assert f(0, P, -4, P, 1, 4, 8, 1.0, P, None) == 1 and f(0, P, 4, P, 1, 2 ** 60, 8, 1.0, P, None) == 1
    assert g(0, P, P, P, P, 4, -1, 8, 1.0, P, P, 1 << 20, None) == 1
    assert lib.euc_codebook_grad_workspace_bytes(0, 0, 8) == 0
    assert lib.euc_codebook_grad_workspace_bytes(8, 10, 8) == 0
    if NO_GPU:
        assert f(0, P, 4, P, 1, 4, 8, 1.0, P, None) == 8
        assert g(0, P, P, P, P, 4, 4, 8, 1.0, P, P, 1 << 20, None) == 8
    else:
        assert f(0, None, 4, P, 1, 4, 8, 1.0, P, None) == 7
        assert g(0, P, P, P, P, 4, 4, 8, 1.0, P, P, 16, None) == 6
        off = ctypes.c_void_p(258)
        assert f(2, P, 4, off, 0, 4, 8, 1.0, P, None) == 7
        assert g(2, P, P, P, P, 4, 4, 8, 1.0, P, off, 1 << 20, None) == 7
        assert g(2, P, P, off, P, 4, 4, 8, 1.0, P, P, 1 << 20, None) == 7
