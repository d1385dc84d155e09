"""Limits of the label operators' arguments that the C ABI checks before it looks for a device."""
import ctypes

import pytest
import torch

NO_GPU = not torch.cuda.is_available()
P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    import _lib
    return _lib.lib()


# fp32, fp64, fp16, bf16: the smallest and largest power of two
@pytest.mark.parametrize("row_type,least,most", [(0, -120, 126), (1, -1014, 1022), (2, -126, 126), (3, -120, 126)])
def test_scales(lib, row_type, least, most):
    def forward(scale, n=0 if not NO_GPU else 4):
        return lib.euc_label_log_probs(row_type, P, 8, n, 8, P, 1, scale, 0, None, None, None, None, None, None)

    def grad(scale, n=0 if not NO_GPU else 4):
        return lib.euc_label_log_probs_grad(row_type, P, 8, n, 8, P, 1, scale, P, P, None, P, None)
    fine = 8 if NO_GPU else 0  # no device, or no rows
    for f in (forward, grad):
        for sign in (1.0, -1.0):
            assert f(sign * 2.0 ** least) == fine and f(sign * 2.0 ** most) == fine
            assert f(sign * 2.0 ** (least - 1)) == 7
            assert f(sign * 2.0 ** (most + 1)) == 7
