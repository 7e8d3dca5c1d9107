"""Layer norm at the ends of its range: workspaces, rows of large values, rows that share 16 bytes."""
import ctypes

import pytest
import torch

import flashinfer_b200 as fb
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", [640, 2048, 3000, 3001, 7168, 16384])
def test_constant_rows_of_large_values_are_the_bias(H, dtype):
    """Values whose square passes fp32's range, in rows of a warp and of a block. With eight significant bits and
    16384 columns at most every sum is exact, so all deviations are zero."""
    x = torch.tensor([2.0 ** 66, 1e20, -1e20, 3e33, -2.0 ** 64], device="cuda").to(torch.bfloat16)
    x = x.to(dtype)[:, None].expand(-1, H).contiguous()
    bias = torch.randn(H, generator=torch.Generator(device="cuda").manual_seed(H), device="cuda").to(dtype)
    h, y = fb.layer_norm(None, x, bias=bias)
    assert h is x and torch.equal(y, bias.expand_as(y))
