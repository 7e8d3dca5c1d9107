"""Layer norm at the ends of its range: workspaces, rows of large values, rows that share 16 bytes."""
import ctypes

import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from tests import layer_refs as R


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


def _rows(H, seed, T=24):
    return torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _place(x, off):
    """x at `off` elements past a 16-byte boundary."""
    buf = torch.zeros(x.numel() + off, dtype=x.dtype, device="cuda")
    buf[off:] = x.reshape(-1)
    return buf[off:].view(x.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("H", [100, 640, 1021, 2048, 3000, 3001, 7168, 16384])
def test_constant_rows_of_any_value_are_the_bias(H, off):
    """The sum of equal values rounds, and so does its quotient: by k units of the value's last place, k at most
    54. The deviations from it are k units exactly, their mean is within 50 * 2^-24 of k units, and added to the
    first mean it rounds to the value."""
    v = torch.tensor([1e20, 1234.567, 1e6 + 0.5, -0.1, 1.0 / 3, 77777.7, -1e-3, 16777215.0], device="cuda")
    x = _place(v[:, None].expand(-1, H), off)
    bias = _rows(H, H, 1)[0]
    _, y = fb.layer_norm(None, x, bias=bias)
    assert torch.equal(y, bias.expand_as(y))


@pytest.mark.gpu
@pytest.mark.parametrize("mean", [5e3, -1e5, 1e6])
@pytest.mark.parametrize("H", [100, 640, 1021, 3000, 3001, 7168, 16384])
def test_rows_with_a_mean_far_above_their_deviations(H, mean):
    """The first mean is off by e0 <= 54 U mean|h| (32 values in a thread, 5 + 5 levels, the quotient). The second is
    rounded once, U |mean|, after a sum of deviations with at most 52 roundings. The squares around the first
    mean have 56; the square of the deviations' mean is taken off them."""
    U = 2.0 ** -24
    x = _rows(H, H) + mean
    leaf = x.clone().requires_grad_()
    _, y = fb.layer_norm(None, leaf, eps=1e-5)
    h = x.double()
    m = h.mean(1, keepdim=True)
    c = h - m
    var = c.square().mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + 1e-5)
    e0 = 54 * U * h.abs().mean(1, keepdim=True)
    dev = c.abs().mean(1, keepdim=True) + e0
    e_mean = U * (m.abs() + e0) + 52 * U * dev
    e_var = 56 * U * (var + e0.square()) + 104 * U * e0 * dev + (52 * U * dev).square() + 3 * U * e0.square()
    rel = e_var / (var + 1e-5) / 2
    rel = rel + 2 * rel.square() + 5 * U
    n = c * r
    en = r * (e_mean + U * (c.abs() + e_mean)) * (1 + rel) + n.abs() * (rel + U)
    R.check(y.detach(), n, en, "normed")
    # the backward pass goes from the same mean and 1 / sqrt(var + eps)
    dy = _rows(H, H + 1)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    u = dy.double()
    s1, s2 = u.mean(1, keepdim=True), (u * n).mean(1, keepdim=True)
    e1 = 61 * U * u.abs().mean(1, keepdim=True)
    e2 = 62 * U * (u * n).abs().mean(1, keepdim=True) + (u.abs() * en).mean(1, keepdim=True)
    mag = r * (u.abs() + s1.abs() + (n * s2).abs())
    ex = r * (e1 + n.abs() * e2 + en * (s2.abs() + e2)) + mag * (rel + 8 * U)
    R.check(dx, r * (u - s1 - n * s2), ex, "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H", [(3000, 3001), (2999, 2050), (1500, 7001), (5000, 515)])
def test_in_place_with_many_rows_that_share_16_bytes(T, H, dtype):
    """hidden over the residual in rows off the 16-byte boundary, far more than there are blocks: neighbouring rows are
    read by one block while another rewrites them. The same bits as into a new tensor, run after run."""
    x, f = (_rows(H, s, T).to(dtype) for s in (1, 2))
    w, b = (_rows(H, s, 1)[0].to(dtype) for s in (3, 4))
    h_ref, y_ref = fb.layer_norm(f, x, weight=w, bias=b)
    for _ in range(5):
        mine = x.clone()
        h, y = fb.layer_norm(f, mine, weight=w, bias=b, output=mine)
        assert h is mine and torch.equal(h, h_ref) and torch.equal(y, y_ref)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [128, 640, 3000, 3001, 7168])
def test_rows_beyond_fp32(H):
    """Deviations whose square is infinite, a sum that is, and an ordinary row between them."""
    x = _rows(H, H, 5)
    x[0] = 2.0 ** 64
    x[0, ::2] = -2.0 ** 64
    x[2, 3] = 2.0 ** 65
    x[4] = torch.finfo(torch.float32).max
    bias = _rows(H, H + 1, 1)[0]
    _, y = fb.layer_norm(None, x, bias=bias)
    assert torch.equal(y[[0, 2]], bias.expand(2, H)) and bool(torch.isnan(y[4]).all())
    _, alone = fb.layer_norm(None, x[[1, 3]], bias=bias)
    R.check(y[[1, 3]], alone.double(), 100 * R.U * (alone.double().abs() + 1), "ordinary rows")
