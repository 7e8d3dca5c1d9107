"""4-bit weights at the ends of their types' ranges, against arithmetic in 64 bits."""
import pytest
import torch

import flashinfer_b200 as fb
from tests import layer_refs as R

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


@pytest.mark.gpu
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("M,E", [(8, 0), (16, 0), (17, 0), (130, 0), (300, 0), (32, 4), (33, 4), (900, 3)])
def test_fp16_scales_far_apart(M, E, f32):
    """One group with scales around 2^8, where the tokens are zero, beside groups of scales down to 2^-30 of them.

    Few rows: the weights are exact, a sum of K products and of the groups' has at most K + 40 roundings. Tensor
    cores: a row's largest scale is moved to [2^9, 2^10). There a weight is off by half a step of fp16, with an fp32
    scale by what its low part's product adds, 2^-7 of that, or by fp16's last step: 15 times 2^-25 of the scale, 2^-25
    each of the product(s): 17 * 2^-25, below 2^-29 of the largest scale."""
    g = torch.Generator(device="cuda").manual_seed(M + E)
    N, K, group = 70, 320, 64
    rows = (E, N) if E else (N,)
    packed = torch.randint(0, 256, (*rows, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    zero = torch.randint(0, 16, (*rows, K // group), generator=g, device="cuda", dtype=torch.uint8)
    far = torch.arange(K // group, device="cuda") > 0
    for down in (10, 16, 20, 22, 24, 27, 30):
        p = torch.where(far, 8.0 - down, 8.0) + torch.rand(*rows, K // group, generator=g, device="cuda")
        scale = torch.exp2(p) if f32 else torch.exp2(p).half()
        x = (256.0 * torch.randn(M, K, generator=g, device="cuda")).half()
        x[:, :group] = 0
        w = (_unpack(packed) - zero.double().repeat_interleave(group, -1)) * scale.double().repeat_interleave(group, -1)
        half, u = 2.0 ** -11, 2.0 ** -24
        if E:
            count = torch.full((E,), M // E)
            count[0] += M - M // E * E
            base = torch.cat([torch.zeros(1), count.cumsum(0)]).int().cuda()
            y = fb.int4_expert_matmul(x, packed, scale, base, zero, group=group)
            parts = [(slice(int(base[e]), int(base[e + 1])), w[e], scale[e]) for e in range(E)]
        else:
            y = fb.int4_matmul(x, packed, scale, zero, group=group)
            parts = [(slice(0, M), w, scale)]
        exact = M <= (8 * E if E else 16)
        for at, we, se in parts:
            xd = x[at].double()
            mag = xd.abs() @ we.abs().t()
            err = mag * (K + 40) * u
            if not exact:
                err = err + mag * half * (1 + 2.0 ** -7)
                err = err + 2.0 ** -29 * xd.abs().sum(1, keepdim=True) * se.double().amax(-1)
            R.check(y[at], xd @ we.t(), err, (down, exact))
