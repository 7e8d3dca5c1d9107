"""4-bit weights: quantisation and back, products dense and per expert, against 64-bit arithmetic."""
import ctypes

import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from tests import layer_refs as R

U = R.U
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def _spread(v, K, group):
    """Per-group values [..., groups] to [..., K]."""
    return v.double()[..., torch.arange(K, device=v.device) // group]


def _weights(packed, scale, zero, group):
    q = _unpack(packed).double()
    K = q.shape[-1]
    z = 8.0 if zero is None else _spread(zero & 15, K, group)
    return (q - z) * _spread(scale, K, group)


# ------------------------------------------------------------------ quantisation
def _quantised(w, group, symmetric):
    """The definition, step by step in fp32 (each an IEEE operation) on the CPU."""
    w = w.cpu()
    K = w.shape[-1]
    n = -(-K // group)
    pad = torch.zeros(*w.shape[:-1], n * group)
    pad[..., :K] = w.float()
    b = pad.view(*w.shape[:-1], n, group)
    least = 2.0 ** -24 if w.dtype == torch.float16 else 2.0 ** -100
    if symmetric:
        step = b.abs().amax(-1) / torch.tensor(7.0)
    else:
        low, high = b.amin(-1).clamp(max=0), b.amax(-1).clamp(min=0)
        step = (high - low) / torch.tensor(15.0)
    scale = step.clamp(min=least).to(w.dtype)
    s = scale.float()
    zero = torch.full_like(s, 8.0) if symmetric else torch.round(-low / s).clamp(0, 15)
    q = torch.round(b / s[..., None]) + zero[..., None]
    q = q.clamp(1 if symmetric else 0, 15).flatten(-2)[..., :K]
    return q.to(torch.uint8), scale, zero.to(torch.uint8)


@pytest.mark.gpu
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape,group", [
    ((1, 32), 32), ((3, 64), 64), ((5, 96), 64), ((2, 160), 128), ((7, 7168), 128), ((130, 256), 32),
    ((3, 2, 544), 256), ((2, 3, 1152), 512), ((9, 1056), 32), ((4, 416), 4096), ((33, 2048), 1024),
    ((2, 800), 384)])
def test_quantise_and_back(shape, group, dtype, symmetric):
    g = _gen(sum(shape) + group)
    w = (torch.randn(*shape, generator=g, device="cuda")
         * torch.exp(torch.randn(*shape[:-1], 1, generator=g, device="cuda"))).to(DT[dtype])
    w[..., 0] = 0
    w.view(-1, shape[-1])[0, :32] = 0          # a group of zeros, or most of one
    packed, scale, zero = fb.quantize_int4(w, group=group, symmetric=symmetric)
    q_ref, s_ref, z_ref = _quantised(w, group, symmetric)
    assert torch.equal(scale.cpu(), s_ref) and torch.equal(_unpack(packed).cpu(), q_ref)
    assert (zero is None) == symmetric
    if not symmetric:
        assert torch.equal(zero.cpu(), z_ref)
    ref = _weights(packed, scale, zero, group)
    for out in (torch.bfloat16, torch.float16, torch.float32):
        back = fb.dequantize_int4(packed, scale, zero, group=group, out_dtype=out)
        assert torch.equal(back, ref.float().to(out))   # q - zero has 5 bits, the product 29: one
        # rounding to fp32 (none for 16-bit scales) and one to the type, as here
    # half a step, and what the rounded scale moves the ends by
    half = torch.finfo(w.dtype).eps / 2
    lim = _spread(scale, shape[-1], group) * (0.5 + 16 * half) + 1e-30
    if not symmetric:
        lim = 2 * lim                                   # the zero point is rounded as well
    assert bool(((ref - w.double()).abs() <= lim + ref.abs() * half).all())


@pytest.mark.gpu
def test_quantise_ties_and_extremes():
    # scale 1: every tie of the range
    row = torch.arange(-14, 15, dtype=torch.float32) / 2
    w = torch.zeros(2, 64)
    w[0, :29] = row
    w[0, 63] = 7.0
    w[1, :29] = row * 2.0 ** -60
    w[1, 63] = 7.0 * 2.0 ** -60
    packed, scale, _ = fb.quantize_int4(w.cuda(), group=64)
    assert torch.equal(scale.cpu(), torch.tensor([[1.0], [2.0 ** -60]]))
    q = torch.round(row) + 8                            # ties to even
    assert torch.equal(_unpack(packed).cpu()[:, :29].float(), q.expand(2, 29))
    tiny = torch.full((1, 32), 2.0 ** -24, dtype=torch.float16, device="cuda")
    packed, scale, _ = fb.quantize_int4(tiny, group=32)
    assert float(scale) == 2.0 ** -24 and bool((_unpack(packed) == 9).all())


@pytest.mark.gpu
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_weights_stay_in_their_group(bad, symmetric):
    w = torch.randn(2, 256, generator=_gen(1), device="cuda", dtype=torch.float32).to(torch.bfloat16)
    clean = w.clone()
    w[1, 70] = bad
    packed, scale, zero = fb.quantize_int4(w, group=64, symmetric=symmetric)
    ref = fb.quantize_int4(clean, group=64, symmetric=symmetric)
    assert not bool(torch.isfinite(scale[1, 1]))
    keep = [0, 2, 3]
    assert torch.equal(scale[1, keep], ref[1][1, keep]) and torch.equal(scale[0], ref[1][0])
    assert torch.equal(_unpack(packed)[1, :64], _unpack(ref[0])[1, :64])
    back = fb.dequantize_int4(packed, scale, zero, group=64)
    assert not bool(torch.isfinite(back[1, 70])) and bool(torch.isfinite(back[0]).all())
    x = torch.ones(1, 256, dtype=torch.bfloat16, device="cuda")
    y = fb.int4_matmul(x, packed, scale, zero, group=64)
    assert bool(torch.isfinite(y[0, 0])) and not bool(torch.isfinite(y[0, 1]))


# ------------------------------------------------------------------ products
def _case(g, M, N, K, group, dtype, zero, f32_scale, E=0):
    shape = (E, N) if E else (N,)
    n = -(-K // group)
    x = torch.randn(M, K, generator=g, device="cuda").to(DT[dtype])
    packed = torch.randint(0, 256, (*shape, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (torch.rand(*shape, n, generator=g, device="cuda") + 0.5) * 0.01
    scale = scale.to(torch.float32 if f32_scale else DT[dtype])
    z = None
    if zero:  # the high half does not count
        z = torch.randint(0, 256, (*shape, n), generator=g, device="cuda", dtype=torch.uint8)
    return x, packed, scale, z


def _product(x, packed, scale, zero, group, bias=None):
    """y and its bound. fp32 products of 16-bit values are exact; a sum of K of them, of the groups'
    products with their scales and of the warps' or parts' shares has at most K + 40 roundings. A weight
    that is rounded to the activations' type is off by half a step of that type, and by the product of a
    fp32 scale's low part that is itself rounded: a 2^-8 of that again. Its error enters as the terms
    themselves do."""
    w = _weights(packed, scale, zero, group)
    xd = x.double()
    y, mag = xd @ w.t(), xd.abs() @ w.abs().t()
    half = torch.finfo(x.dtype).eps / 2
    err = mag * ((x.shape[1] + 40) * U + half * (1 + 2.0 ** -7))
    if bias is not None:
        y = y + bias.double()
        err = err + 4 * U * bias.double().abs()
    return y, err


# one token to many, odd channels, short and ragged depths, groups of every kind
SIZES = [(1, 1, 32, 32), (1, 4096, 7168, 128), (2, 129, 96, 64), (3, 17, 160, 128), (7, 33, 416, 256),
         (8, 64, 1024, 64), (9, 100, 7168, 32), (16, 257, 2048, 128), (17, 48, 544, 32),
         (31, 130, 800, 384), (33, 65, 288, 4096), (64, 2047, 512, 128), (65, 128, 1056, 64),
         (130, 384, 2112, 128), (257, 300, 640, 32), (300, 1000, 1024, 1024), (517, 2047, 1152, 128),
         (1025, 130, 96, 32), (600, 7, 2048, 64), (1, 3, 11776, 128), (4, 5000, 64, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K,group", SIZES)
def test_matmul(M, N, K, group, dtype):
    g = _gen(M + N + K)
    for zero, f32, with_bias in ((False, False, False), (True, True, True), (True, False, False)):
        x, packed, scale, z = _case(g, M, N, K, group, dtype, zero, f32)
        bias = torch.randn(N, generator=g, device="cuda") if with_bias else None
        y = fb.int4_matmul(x, packed, scale, z, bias, group=group)
        assert y.dtype == x.dtype
        R.check(y, *_product(x, packed, scale, z, group, bias), (zero, f32))


def _expert_check(y, x, packed, scale, z, group, base):
    M = x.shape[0]
    most, clean = 0, []
    for b in base.tolist():
        most = max(most, min(max(b, 0), M))
        clean.append(most)
    for e, (lo, hi) in enumerate(zip(clean[:-1], clean[1:])):
        if lo < hi:
            ref, err = _product(x[lo:hi], packed[e], scale[e], None if z is None else z[e], group)
            R.check(y[lo:hi], ref, err, e)
    return clean


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K,group", [
    ([1], 33, 64, 32), ([0, 3, 0, 1], 100, 256, 128), ([5, 0, 20, 7], 257, 416, 64),
    ([130, 1, 0, 300, 17], 200, 1152, 128), ([0, 0, 513], 384, 544, 32), ([2] * 32, 128, 7168, 128),
    ([0, 1] * 128, 40, 128, 64), ([9, 8, 16, 33, 64, 65], 144, 2048, 256)])
def test_expert_matmul(counts, N, K, group, dtype):
    g = _gen(sum(counts) + N + K)
    E, M = len(counts), sum(counts) + 5                 # rows behind the last expert
    base = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    for zero in (False, True):
        x, packed, scale, z = _case(g, M, N, K, group, dtype, zero, zero, E)
        y = fb.int4_expert_matmul(x, packed, scale, base, z, group=group)
        _expert_check(y, x, packed, scale, z, group, base)
        assert not bool(y[sum(counts):].any())
        out = torch.full((M, N), 3.0, dtype=x.dtype, device="cuda")
        got = fb.int4_expert_matmul(x, packed, scale, base, z, group=group, output=out)
        assert got is out and bool((out[sum(counts):] == 3).all())
        assert torch.equal(out[:sum(counts)], y[:sum(counts)])


@pytest.mark.gpu
@pytest.mark.parametrize("base", [[4, 9, 30], [-7, 5, 99], [0, 20, 10, 25], [25, 3, 30], [0, 0, 0, 0]])
@pytest.mark.parametrize("M", [30, 400])
def test_bases_of_any_kind(base, M):
    """Ranges that start late, step back or leave the rows: each row has one expert or none."""
    g = _gen(5)
    base = torch.tensor([b * M // 30 for b in base], dtype=torch.int32, device="cuda")
    E = base.numel() - 1
    x, packed, scale, z = _case(g, M, 72, 320, 64, "bf16", True, False, E)
    y = fb.int4_expert_matmul(x, packed, scale, base, z, group=64)
    clean = _expert_check(y, x, packed, scale, z, 64, base)
    assert not bool(y[:clean[0]].any()) and not bool(y[clean[-1]:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 70, 300])
def test_far_scales_and_values(M):
    """Scales from 2^-70 to 2^40 (bf16) and into fp16's subnormals, in one row and in different ones."""
    g = _gen(M)
    x, packed, scale, z = _case(g, M, 90, 512, 64, "bf16", True, False)
    p = torch.randint(-70, 41, (90, 8), generator=g, device="cuda")
    scale = torch.ldexp(torch.ones(90, 8, device="cuda"), p).to(torch.bfloat16)
    R.check(fb.int4_matmul(x, packed, scale, z, group=64), *_product(x, packed, scale, z, 64), "bf16")
    x, packed, _, z = _case(g, M, 90, 512, 64, "fp16", True, False)
    for f32 in (False, True):
        p = torch.randint(-24, -8, (90, 8), generator=g, device="cuda")
        scale = torch.ldexp(torch.ones(90, 8, device="cuda"), p).to(
            torch.float32 if f32 else torch.float16)
        R.check(fb.int4_matmul(x, packed, scale, z, group=64), *_product(x, packed, scale, z, 64), f32)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 300])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_non_finite_tokens_stay_in_their_row(M, dtype):
    g = _gen(3)
    x, packed, scale, z = _case(g, M, 100, 288, 32, dtype, True, False)
    x[1, 7], x[3, 200] = float("nan"), float("inf")
    y = fb.int4_matmul(x, packed, scale, z, group=32)
    ref = x.double() @ _weights(packed, scale, z, 32).t()
    assert bool(torch.isnan(y[1]).all())
    assert torch.equal(torch.isnan(y[3]), torch.isnan(ref[3]))
    assert torch.equal(y[3][~torch.isnan(y[3])].double(), ref[3][~torch.isnan(ref[3])])
    rest = [i for i in range(M) if i not in (1, 3)]
    assert bool(torch.isfinite(y[rest]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 12, 100, 700])
def test_same_bits_again_on_another_stream_and_in_a_graph(M):
    g = _gen(M)
    x, packed, scale, z = _case(g, M, 640, 1056, 32, "bf16", True, False)
    first = fb.int4_matmul(x, packed, scale, z, group=32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [fb.int4_matmul(x, packed, scale, z, group=32) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, y) for y in again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fb.int4_matmul(x, packed, scale, z, group=32)
    x.copy_(torch.randn(M, 1056, generator=g, device="cuda"))
    graph.replay()
    assert torch.equal(y, fb.int4_matmul(x, packed, scale, z, group=32))


@pytest.mark.gpu
def test_no_rows_and_odd_outputs():
    x, packed, scale, _ = _case(_gen(0), 0, 16, 64, 32, "fp16", False, False)
    assert fb.int4_matmul(x, packed, scale, group=32).shape == (0, 16)
    w = torch.zeros((0, 64), device="cuda")
    p, s, _ = fb.quantize_int4(w, group=32)
    assert p.shape == (0, 32) and fb.dequantize_int4(p, s, group=32).shape == (0, 64)
    for M in (3, 100, 300):
        x, packed, scale, _ = _case(_gen(1), M, 33, 64, 32, "fp16", False, False)
        buf = torch.zeros(M * 33 + 1, dtype=torch.float16, device="cuda")
        out = buf[1:].view(M, 33)
        fb.int4_matmul(x, packed, scale, group=32, output=out)
        assert torch.equal(out, fb.int4_matmul(x, packed, scale, group=32)) and float(buf[0]) == 0


@pytest.mark.gpu
def test_quantised_weights_in_a_product():
    """The format that the quantiser writes is the one that the products read."""
    g = _gen(4)
    for dtype, sym in ((torch.bfloat16, True), (torch.float16, False)):
        w = (torch.randn(200, 640, generator=g, device="cuda") * 0.05).to(dtype)
        packed, scale, zero = fb.quantize_int4(w, group=64, symmetric=sym)
        wd = fb.dequantize_int4(packed, scale, zero, group=64, out_dtype=torch.float32).double()
        for M in (2, 150):
            x = torch.randn(M, 640, generator=g, device="cuda").to(dtype)
            y = fb.int4_matmul(x, packed, scale, zero, group=64)
            ref, err = _product(x, packed, scale, zero, 64)
            assert bool(((x.double() @ wd.t() - ref).abs() <= 1e-9 + 2 * U * err / U).all())
            R.check(y, ref, err, M)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, packed, scale, z = _case(_gen(0), 4, 16, 128, 64, "bf16", True, False)
    with pytest.raises(TypeError, match="x must be"):
        fb.int4_matmul(x.float(), packed, scale, z, group=64)
    with pytest.raises(TypeError, match="weight"):
        fb.int4_matmul(x, packed.to(torch.int8), scale, z, group=64)
    with pytest.raises(ValueError, match="do not fit"):
        fb.int4_matmul(x, packed[:, :32].contiguous(), scale, z, group=64)
    with pytest.raises(ValueError, match="scale must have shape"):
        fb.int4_matmul(x, packed, scale, z, group=32)
    with pytest.raises(TypeError, match="scale"):
        fb.int4_matmul(x, packed, scale.half(), z, group=64)
    with pytest.raises(TypeError, match="zero"):
        fb.int4_matmul(x, packed, scale, z.int(), group=64)
    for group in (0, 16, 96, 129, -128):
        with pytest.raises(ValueError, match="group"):
            fb.int4_matmul(x, packed, scale, z, group=group)
    with pytest.raises(ValueError, match="multiple of 32"):
        fb.quantize_int4(torch.zeros((2, 48), device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        fb.int4_matmul(x, packed, scale, z, torch.zeros(15, device="cuda"), group=64)
    with pytest.raises(ValueError, match="no gradient"):
        fb.int4_matmul(x.clone().requires_grad_(), packed, scale, z, group=64)
    with pytest.raises(ValueError, match="no gradient"):
        fb.quantize_int4(torch.zeros((2, 64), device="cuda", requires_grad=True))
    with pytest.raises(RuntimeError, match="SHAPE"):    # the output over x
        fb.int4_matmul(x, packed, scale, z, group=64, output=x.view(-1)[:64].view(4, 16))
    with pytest.raises(RuntimeError, match="ALIGN"):
        buf = torch.zeros(4 * 128 + 1, dtype=torch.bfloat16, device="cuda")
        fb.int4_matmul(buf[1:].view(4, 128), packed, scale, z, group=64)
    e = packed.view(1, 16, 64)
    with pytest.raises(ValueError, match="expert_base"):
        fb.int4_expert_matmul(x, e, scale.view(1, 16, 2), torch.zeros(3, dtype=torch.int32, device="cuda"),
                              group=64)
    with pytest.raises(ValueError, match="do not fit"):
        fb.int4_expert_matmul(x, packed, scale, torch.zeros(2, dtype=torch.int32, device="cuda"))
    out = torch.zeros((4, 16), dtype=torch.bfloat16, device="cuda")
    version = out._version
    fb.int4_matmul(x, packed, scale, z, group=64, output=out)
    assert out._version > version


def test_refusals_on_the_host():
    with pytest.raises(ValueError, match="CUDA"):
        fb.quantize_int4(torch.zeros((2, 64)))
    with pytest.raises(ValueError, match="CUDA"):
        fb.dequantize_int4(torch.zeros((2, 64), dtype=torch.uint8), torch.zeros((2, 1)))
    with pytest.raises(ValueError, match="CUDA"):
        fb.int4_matmul(torch.zeros((2, 64), dtype=torch.float16), None, None)
    lib = _lib.load()
    size = ctypes.c_size_t()
    for bad in ((-1, 8, 64, 1), (1, 0, 64, 1), (1, 8, 48, 1), (1, 8, 131104, 1), (1, 8, 64, 257)):
        assert lib.fmoe_int4_workspace_size(*bad, ctypes.byref(size)) == -2, bad
    assert lib.fmoe_int4_workspace_size(1, 8, 64, 1, None) == -1
    assert lib.fmoe_int4_workspace_size(1, 8, 64, 1, ctypes.byref(size)) == 0
    q = lambda w=1 << 20, dtype=1, rows=4, k=64, group=32, packed=2 << 20, scale=3 << 20, zero=None: \
        lib.fmoe_quantize_int4(w, dtype, rows, k, group, packed, scale, zero, None)  # noqa: E731
    assert q(rows=-1) == -2 and q(k=48) == -2 and q(group=0) == -2 and q(group=96) == -2
    assert q(dtype=4) == -6 and q(w=None) == -1 and q(packed=None) == -1 and q(scale=None) == -1
    assert q(w=(1 << 20) + 2) == -3 and q(packed=(2 << 20) + 8) == -3
    assert q(packed=1 << 20) == -2 and q(rows=0) == 0
    d = lambda packed=1 << 20, scale=2 << 20, sd=1, zero=None, rows=4, k=64, group=32, w=3 << 20, dtype=1: \
        lib.fmoe_dequantize_int4(packed, scale, sd, zero, rows, k, group, w, dtype, None)  # noqa: E731
    assert d(rows=-1) == -2 and d(k=0) == -2 and d(group=33) == -2 and d(sd=9) == -6
    assert d(packed=None) == -1 and d(w=(3 << 20) + 4) == -3 and d(w=1 << 20) == -2 and d(rows=0) == 0
    assert lib.fmoe_int4_matmul(None, None) == -1
    a = _lib.FmoeInt4Args()

    def run(**kw):
        a.num_rows, a.n, a.k, a.num_experts, a.group, a.dtype, a.scale_dtype = 4, 16, 64, 1, 32, 1, 1
        a.x, a.weight, a.scale, a.zero = 1 << 20, 2 << 20, 3 << 20, None
        a.bias, a.expert_base, a.out, a.zero_tail = None, None, 4 << 20, 1
        a.workspace, a.workspace_bytes = None, 0
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.fmoe_int4_matmul(ctypes.byref(a), None)
    for bad in ({"num_rows": -1}, {"n": 0}, {"k": 40}, {"k": 131104}, {"group": 48}, {"group": 0},
                {"num_experts": 0}, {"num_experts": 257}, {"out": 1 << 20},
                {"expert_base": 5 << 20, "bias": 6 << 20},
                {"n": 1 << 30, "num_experts": 2, "expert_base": 5 << 20}):
        assert run(**bad) == -2, bad
    assert run(num_experts=2) == -1 and run(x=None) == -1 and run(scale=None) == -1
    assert run(dtype=0, scale_dtype=0) == -6 and run(scale_dtype=2) == -6
    assert run(x=(1 << 20) + 2) == -3 and run(weight=(2 << 20) + 8) == -3 and run(out=(4 << 20) + 1) == -3
    assert run(num_rows=0) == 0
