"""4-bit weights at the ends of their types' ranges, against arithmetic in 64 bits."""
import pytest
import torch

import flashinfer_b200 as fb

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("K,group", [(64, 32), (256, 128), (512, 256), (1024, 512)])
def test_groups_wider_than_the_largest_number(K, group, dtype):
    """Finite weights whose largest less their smallest is beyond fp32: the scale is a fifteenth of it all the same.
    Rounded to the type it is off by half a step; q and the zero point are each off by a half, and at the ends
    by what the rounded scale moves them (16 half steps of the type)."""
    top = torch.finfo(DT[dtype]).max
    w = torch.zeros(5, K, dtype=torch.float64)
    w[0, :2] = torch.tensor([2e38, -2e38])
    w[1, :3] = torch.tensor([3e38, -1e38, 5e37])
    w[2, :3] = torch.tensor([3e37, -3.2e38, 2e37])
    w[3, :2] = torch.tensor([top, -top])
    w[4] = torch.linspace(-1.0, 1.0, K, dtype=torch.float64) * 2.5e38
    w = w.to(DT[dtype])
    packed, scale, zero = (t.cpu() for t in fb.quantize_int4(w.cuda(), group=group, symmetric=False))
    assert bool(torch.isfinite(scale).all())
    b = w.double().view(5, K // group, group)
    low, high = b.amin(2).clamp(max=0), b.amax(2).clamp(min=0)
    half = torch.finfo(DT[dtype]).eps / 2
    exact = ((high - low) / 15).clamp(min=2.0 ** -100)
    # formed in fp32 (three roundings), then rounded to the type
    assert bool(((scale.double() - exact).abs() <= exact * (half + 4 * 2.0 ** -24)).all())
    s = scale.double()
    assert torch.equal(zero.double(), torch.round((-low / s).float()).double().clamp(0, 15))
    back = (_unpack(packed).view_as(b) - zero.double()[:, :, None]) * s[:, :, None]
    assert bool(((back - b).abs() <= s[:, :, None] * (1 + 32 * half)).all())
    # what fits the type comes back as it stands for
    got = fb.dequantize_int4(packed.cuda(), scale.cuda(), zero.cuda(), group=group, out_dtype=DT[dtype]).cpu()
    fits = (back.abs() <= top).view(5, K)
    assert torch.equal(got[fits], back.view(5, K).float().to(DT[dtype])[fits])
    assert bool(torch.isfinite(got[:3]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_wide_group_with_an_infinity_or_a_nan(bad):
    w = torch.full((2, 64), 3e38, device="cuda")
    w[:, ::2] = -3e38
    w[0, 5] = bad
    _, scale, _ = fb.quantize_int4(w, group=64, symmetric=False)
    assert not bool(torch.isfinite(scale[0])) and bool(torch.isfinite(scale[1]))
