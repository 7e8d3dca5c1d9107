"""Layer norm at the ends of its range: workspaces, rows of large values, rows that share 16 bytes."""
import ctypes

import pytest
import torch  # noqa: F401  (its libraries before the package's)

from flashinfer_b200 import _lib


@pytest.mark.parametrize("off", [4, 8, 12])
def test_a_workspace_off_the_16_byte_boundary_is_refused(off):
    """Pairs and fours of the sums over rows go through it. Checked on the host, before any launch."""
    back = _lib.load().fmoe_layer_norm_backward
    need = 2 * 4 * 1024 * 4
    a = _lib.FmoeLayerNormArgs(num_tokens=4, hidden_size=1024, dtype=1, branch=1 << 20,
                               residual=2 << 20, weight=3 << 20, bias=4 << 20, weight_dtype=1,
                               bias_dtype=1, eps=1e-5, stats=5 << 20, grad_normed=6 << 20,
                               workspace=(8 << 20) + off, workspace_bytes=need)
    for field in ("grad_weight", "grad_bias"):
        a.grad_weight = a.grad_bias = None
        setattr(a, field, 7 << 20)
        assert back(ctypes.byref(a), None) == -3, field
    # one that no sum needs is not looked at: the next check answers (the input gradient over the residual)
    a.grad_weight = a.grad_bias = None
    a.grad_input = 2 << 20
    assert back(ctypes.byref(a), None) == -2
