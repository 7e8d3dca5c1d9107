"""Layer norm with the residual sum, forward and backward, against its definition in 64 bits."""
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


def _inputs(T, H, dtype, branch, weight, bias, f32=False, seed=0, off=0):
    """Rows of a few units around a mean of their own; off: elements past a 16-byte boundary."""
    g = _gen(seed + T + H)
    par = torch.float32 if f32 else dtype

    def place(v, t):
        buf = torch.zeros(v.numel() + off, dtype=t, device="cuda")
        buf[off:] = v.reshape(-1)
        return buf[off:].view(v.shape)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = place(2 * rand(T, H) + 3 * rand(T, 1), dtype)
    f = place(rand(T, H), dtype) if branch else None
    w = place(1 + 0.3 * rand(H), par) if weight else None
    b = place(0.5 * rand(H), par) if bias else None
    return f, x, w, b


def _ref(f, x, w, b, eps):
    """hidden, normed, n, r, and the bounds of normed and of n and the relative one of r.

    The mean is a sum of H terms: at most 32 in a thread, 5 shuffle levels, 16 warps and a product:
    54 roundings, off by em = 54 U mean|h|. A deviation is off by em, the rounding of h and its own.
    The errors of the mean cancel in the sum of squares to first order (the deviations add up to
    zero), which leaves em^2, the other roundings, and 64 roundings of the sum and the warps' joining,
    in which a warp's own mean is off by 40 U mean|h| and, like em, enters squared. rsqrtf is within
    two units in the last place (4 U), the sum with eps U.
    """
    h = x.double() if f is None else x.double() + f.double()
    H = h.shape[1]
    mean = h.mean(1, keepdim=True)
    c = h - mean
    var = c.square().mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    em = 54 * U * h.abs().mean(1, keepdim=True)
    ec = em + U * h.abs() + U * c.abs()
    rel_var = (64 * U * var + (2 * c.abs() * (U * h.abs() + U * c.abs())).mean(1, keepdim=True)
               + 2 * em.square() + ec.square().mean(1, keepdim=True)) / (var + eps)
    rel_r = rel_var / 2 + 5 * U
    n = c * r
    en = r * ec + n.abs() * (rel_r + U)
    wd = torch.ones(H, dtype=torch.float64, device=x.device) if w is None else w.double()
    y = n * wd
    ey = wd.abs() * en + U * y.abs()
    if b is not None:
        y = y + b.double()
        ey = ey + U * y.abs()
    return h, y, n, r, ey, en, rel_r, wd


CASES = [  # T, H, dtype, branch, weight, bias, fp32 parameters
    (1, 1, "fp32", False, True, True, False), (3, 2, "bf16", True, True, True, False),
    (1, 7168, "bf16", True, True, True, False), (16, 7168, "bf16", False, True, False, True),
    (5, 33, "fp16", True, True, True, True), (9, 128, "bf16", True, False, True, False),
    (300, 512, "bf16", True, True, True, False), (257, 520, "fp16", True, True, False, False),
    (600, 1024, "fp32", True, True, True, False), (77, 1032, "bf16", True, True, True, True),
    (13, 1025, "bf16", True, True, True, False), (500, 4096, "bf16", True, True, True, False),
    (450, 2047, "fp16", True, True, True, False), (3, 8192, "fp32", True, True, True, False),
    (7, 8200, "bf16", True, True, True, False), (160, 9001, "fp16", False, True, True, True),
    (4, 16384, "fp32", True, True, True, False), (5, 16384, "bf16", True, False, False, False),
    (2, 16383, "fp32", True, True, True, False), (40, 64, "fp32", False, False, False, False)]


def _grads_ref(f, x, w, b, dh, dy, eps):
    """The formula's gradients and their bounds.

    u = dy w is rounded once; the row sums of u and u n have at most 60 roundings of their own (16 or 32
    values in a thread, 5 levels, 16 warps, a product), u n in addition n's error. Then three operations on
    the way out. Sums over rows: a thread's rows, eight warps, and the blocks in eight parts: at most
    T + 40 additions, each product with n's error.
    """
    h, _, n, r, _, en, rel_r, wd = _ref(f, x, w, b, eps)
    T, H = h.shape
    zero = torch.zeros_like(h)
    dh = zero if dh is None else dh.double()
    dy = zero if dy is None else dy.double()
    u = dy * wd
    s1, s2 = u.mean(1, keepdim=True), (u * n).mean(1, keepdim=True)
    e1 = 61 * U * u.abs().mean(1, keepdim=True)
    e2 = 62 * U * (u * n).abs().mean(1, keepdim=True) + (u.abs() * en).mean(1, keepdim=True)
    dx = dh + r * (u - s1 - n * s2)
    mag = r * (u.abs() + s1.abs() + (n * s2).abs())
    ex = r * (e1 + n.abs() * e2 + en * s2.abs()) + mag * (rel_r + 6 * U) + 2 * U * (dh.abs() + mag)
    out = {"x": (dx, ex)}
    out["w"] = ((dy * n).sum(0), ((T + 40) * U * (dy * n).abs() + dy.abs() * en).sum(0))
    out["b"] = (dy.sum(0), ((T + 40) * U * dy.abs()).sum(0))
    return out


def _check_all(f, x, w, b, eps, seed=3, drop=None):
    T, H = x.shape
    g = _gen(seed)
    h_ref, y_ref, _, _, ey, _, _, _ = _ref(f, x, w, b, eps)
    eh = U * h_ref.abs() if f is not None else torch.zeros_like(h_ref)
    h, y = fb.layer_norm(f, x, weight=w, bias=b, eps=eps)
    R.check(h, h_ref, eh, "hidden")
    R.check(y, y_ref, ey, "normed")
    leaves = [t for t in (f, x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_()
    h, y = fb.layer_norm(f, x, weight=w, bias=b, eps=eps)
    R.check(h.detach(), h_ref, eh, "hidden, recorded")
    R.check(y.detach(), y_ref, ey, "normed, recorded")
    dh = None if drop == "hidden" else torch.randn(T, H, generator=g, device="cuda").to(x.dtype)
    dy = None if drop == "normed" else torch.randn(T, H, generator=g, device="cuda").to(x.dtype)
    pairs = [(o, d) for o, d in ((h, dh), (y, dy)) if d is not None]
    got = torch.autograd.grad([o for o, _ in pairs], leaves, [d for _, d in pairs])
    for t in leaves:
        t.requires_grad_(False)
    ref = _grads_ref(f, x, w, b, dh, dy, eps)
    names = [n for n, t in (("f", f), ("x", x), ("w", w), ("b", b)) if t is not None]
    for name, d in zip(names, got):
        R.check(d, *ref["x" if name == "f" else name], "d " + name)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,dtype,branch,weight,bias,f32", CASES)
def test_forward_and_gradients(T, H, dtype, branch, weight, bias, f32):
    _check_all(*_inputs(T, H, DT[dtype], branch, weight, bias, f32), 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("H,dtype", [(200, "bf16"), (1160, "fp16"), (2052, "fp32"), (8448, "bf16")])
def test_off_the_16_byte_boundary(H, dtype):
    f, x, w, b = _inputs(11, H, DT[dtype], True, True, True, off=1)
    assert x.data_ptr() % 16 != 0
    _check_all(f, x, w, b, 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("drop", ["hidden", "normed"])
@pytest.mark.parametrize("H", [96, 1536])
def test_one_gradient_alone(H, drop):
    _check_all(*_inputs(21, H, torch.bfloat16, True, True, True), 1e-5, drop=drop)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [40, 2000])
def test_many_rows_per_block(H):
    """More rows than blocks, by far: every row once, and the sums over all of them."""
    T = 5000 if H == 40 else 3001
    f, x, w, b = _inputs(T, H, torch.float32, True, True, True)
    _check_all(f, x, w, b, 1e-5)


@pytest.mark.gpu
def test_large_mean_and_constant_rows():
    x = torch.randn(6, 1000, generator=_gen(1), device="cuda") + 4096.0
    _check_all(None, x, None, None, 0.0)
    c = torch.full((3, 1000), 3.0, device="cuda")
    c[1] = 0
    _, y = fb.layer_norm(None, c, eps=1e-5)
    assert not bool(y.any())
    bias = torch.arange(1000.0, device="cuda")
    _, y = fb.layer_norm(None, c, bias=bias)
    assert torch.equal(y, bias.expand(3, 1000))


@pytest.mark.gpu
@pytest.mark.parametrize("H", [64, 3000])
def test_non_finite_rows_stay_in_their_row(H):
    f, x, w, b = _inputs(5, H, torch.float16, True, True, True)
    x[1, 3], f[3, 7] = float("nan"), float("inf")
    h, y = fb.layer_norm(f, x, weight=w, bias=b)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[3]).all())
    assert bool(torch.isinf(h[3, 7])) and bool(torch.isfinite(y[[0, 2, 4]]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,dtype,branch", [(1, 128, "bf16", True), (16, 7168, "bf16", True),
                                              (5, 1280, "fp16", False), (700, 2048, "bf16", True),
                                              (9, 256, "fp32", True), (2000, 1152, "fp32", False)])
def test_quantised_output(T, H, dtype, branch):
    f, x, w, b = _inputs(T, H, DT[dtype], branch, True, True)
    _, y_ref, _, _, ey, _, _, _ = _ref(f, x, w, b, 1e-5)
    h, (q, scale) = fb.layer_norm(f, x, weight=w, bias=b, quantize=True)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (H // 128, T)
    blocks, bounds = y_ref.view(T, H // 128, 128), ey.view(T, H // 128, 128)
    amax, e_max = blocks.abs().amax(2), bounds.amax(2)
    s = scale.t().double()
    # the largest value within its bound, one division
    assert bool(((s - amax / 448).abs() <= e_max / 448 + U * (amax + e_max) / 448).all())
    back = q.double().view(T, H // 128, 128) * s[:, :, None]
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below its smallest normal number
    v = blocks.abs() + bounds
    lim = bounds + torch.maximum(v * 2.0 ** -4, s[:, :, None] * 2.0 ** -10) + 2 * U * v
    assert bool(((back - blocks).abs() <= lim).all())
    if f is None:
        assert h is x


@pytest.mark.gpu
def test_in_place_and_given_output():
    f, x, w, b = _inputs(9, 640, torch.bfloat16, True, True, True)
    h_ref, y_ref = fb.layer_norm(f, x, weight=w, bias=b)
    keep = x.clone()
    h, y = fb.layer_norm(f, keep, weight=w, bias=b, output=keep)
    assert h is keep and torch.equal(keep, h_ref) and torch.equal(y, y_ref)
    out = torch.full_like(x, 7)
    h, y = fb.layer_norm(None, x, weight=w, bias=b, output=out)
    assert h is out and torch.equal(out, x)


@pytest.mark.gpu
def test_no_tokens():
    x = torch.zeros((0, 256), device="cuda", requires_grad=True)
    w = torch.ones(256, device="cuda", requires_grad=True)
    b = torch.ones(256, device="cuda", requires_grad=True)
    h, y = fb.layer_norm(None, x, weight=w, bias=b)
    assert h.shape == y.shape == (0, 256)
    dx, dw, db = torch.autograd.grad((h.sum() + y.sum()), (x, w, b))
    assert dx.shape == (0, 256) and not bool(dw.any()) and not bool(db.any())


@pytest.mark.gpu
def test_same_bits_again_and_on_another_stream():
    f, x, w, b = (t.requires_grad_() for t in _inputs(999, 1408, torch.bfloat16, True, True, True))
    d = torch.randn(999, 1408, generator=_gen(0), device="cuda").to(torch.bfloat16)

    def step():
        h, y = fb.layer_norm(f, x, weight=w, bias=b)
        return [h.detach(), y.detach(), *torch.autograd.grad((h, y), (f, x, w, b), (d, d))]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.gpu
def test_gradients_against_differences():
    """d loss along a direction against the difference quotient of the 64-bit definition."""
    T, H, eps = 5, 96, 1e-5
    f, x, w, b = (t.requires_grad_() for t in _inputs(T, H, torch.float32, True, True, True))
    g = _gen(9)
    a, c = (torch.randn(T, H, generator=g, device="cuda") for _ in range(2))
    h, y = fb.layer_norm(f, x, weight=w, bias=b, eps=eps)
    grads = torch.autograd.grad((h, y), (f, x, w, b), (a, c))

    def loss(tensors):
        hh, yy = _ref(*tensors, eps)[:2]
        return (hh * a.double()).sum() + (yy * c.double()).sum()
    base = [t.detach().double() for t in (f, x, w, b)]
    for i, d in enumerate(grads):
        way = torch.randn(base[i].shape, generator=g, device="cuda").double()
        step = 1e-6
        lo, hi = list(base), list(base)
        hi[i], lo[i] = base[i] + step * way, base[i] - step * way
        quotient = (loss(hi) - loss(lo)) / (2 * step)
        got = (d.double() * way).sum()
        # fp32 gradients: 1e-5 of the terms' magnitudes; the quotient's own error is of order 1e-9
        assert abs(float(got - quotient)) <= 1e-5 * float((d.double() * way).abs().sum()) + 1e-6


@pytest.mark.gpu
def test_hidden_of_no_branch_is_the_residual():
    x = torch.randn(4, 64, generator=_gen(0), device="cuda")
    h, _ = fb.layer_norm(None, x)
    assert h is x
    leaf = x.clone().requires_grad_()
    h, y = fb.layer_norm(None, leaf)
    assert h.data_ptr() == leaf.data_ptr()
    (d,) = torch.autograd.grad(h.sum(), leaf)
    assert torch.equal(d, torch.ones_like(d))


@pytest.mark.gpu
def test_a_captured_training_step():
    f, x, w, b = (t.requires_grad_() for t in _inputs(33, 384, torch.bfloat16, True, True, True))
    d = torch.randn(33, 384, generator=_gen(5), device="cuda").to(torch.bfloat16)

    def step():
        h, y = fb.layer_norm(f, x, weight=w, bias=b)
        return [y.detach(), *torch.autograd.grad((h, y), (f, x, w, b), (d, d))]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn(33, 384, generator=_gen(6), device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, step()))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    f, x, w, b = _inputs(4, 64, torch.bfloat16, True, True, True)
    with pytest.raises(TypeError, match="branch"):
        fb.layer_norm(f.float(), x)
    with pytest.raises(ValueError, match="branch"):
        fb.layer_norm(f[:3], x)
    with pytest.raises(TypeError, match="weight"):
        fb.layer_norm(f, x, weight=w.half())
    with pytest.raises(ValueError, match="bias"):
        fb.layer_norm(f, x, bias=b[:32])
    with pytest.raises(ValueError, match="contiguous"):
        fb.layer_norm(f, x.t().contiguous().t())
    with pytest.raises(ValueError, match="hidden size"):
        fb.layer_norm(None, torch.zeros((1, 16385), device="cuda"))
    with pytest.raises(ValueError, match="multiple of 128"):
        fb.layer_norm(f, x, quantize=True)
    with pytest.raises(ValueError, match="eps"):
        fb.layer_norm(f, x, eps=float("nan"))
    with pytest.raises(ValueError, match="no gradient"):
        fb.layer_norm(None, torch.zeros((1, 128), device="cuda", requires_grad=True), quantize=True)
    with pytest.raises(ValueError, match="gradients"):
        fb.layer_norm(f.clone().requires_grad_(), x, output=torch.empty_like(x))
    with pytest.raises(RuntimeError, match="SHAPE"):   # the output overlaps the branch
        fb.layer_norm(f, x, output=f)
    with pytest.raises(RuntimeError, match="ALIGN"):
        t = torch.zeros(129, dtype=torch.bfloat16, device="cuda")[1:].view(1, 128)
        fb.layer_norm(None, t, quantize=True)
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(fb.layer_norm(f, leaf)[1].sum(), leaf, create_graph=True)


def test_refusals_on_the_host():
    with pytest.raises(ValueError, match="CUDA"):
        fb.layer_norm(None, torch.zeros((2, 8)))
    lib = _lib.load()
    size = ctypes.c_size_t()
    assert lib.fmoe_layer_norm_workspace_size(5, 64, ctypes.byref(size)) == 0
    assert size.value == 2 * 5 * 64 * 4
    assert lib.fmoe_layer_norm_workspace_size(5, 16385, ctypes.byref(size)) == -2
    assert lib.fmoe_layer_norm_workspace_size(5, 64, None) == -1
    assert lib.fmoe_layer_norm(None, None) == -1
    a = _lib.FmoeLayerNormArgs()

    def run(fn=lib.fmoe_layer_norm, **kw):
        for k in ("hidden", "normed", "normed_q", "normed_scale", "stats", "grad_hidden",
                  "grad_normed", "grad_input", "grad_weight", "grad_bias", "workspace"):
            setattr(a, k, None)
        a.workspace_bytes = 0
        a.num_tokens, a.hidden_size, a.dtype, a.eps = 4, 128, 1, 1e-5
        a.branch, a.residual, a.weight, a.bias = 1 << 20, 2 << 20, 3 << 20, None
        a.weight_dtype = a.bias_dtype = 1
        for k, v in kw.items():
            setattr(a, k, v)
        return fn(ctypes.byref(a), None)
    back = lib.fmoe_layer_norm_backward
    assert run(hidden_size=0) == -2 and run(hidden_size=16385) == -2 and run(num_tokens=-1) == -2
    assert run(dtype=5) == -6 and run(weight_dtype=2) == -6
    assert run(residual=None) == -1
    assert run(residual=(2 << 20) + 1) == -3 and run(stats=(9 << 20) + 4) == -3
    assert run(normed=5 << 20, normed_q=6 << 20) == -2
    assert run(normed_q=6 << 20) == -1                                  # no scales
    assert run(normed_q=6 << 20, normed_scale=7 << 20, hidden_size=130) == -2
    assert run(normed_q=(6 << 20) + 8, normed_scale=7 << 20) == -3
    assert run(hidden=1 << 20) == -2                                    # hidden over the branch
    assert run(normed=(2 << 20) + 256) == -2                            # normed over the residual
    assert run(num_tokens=0) == 0 and run() == 0                        # nothing to write
    assert run(back) == 0
    assert run(back, grad_input=5 << 20) == -1                          # no stats
    assert run(back, grad_bias=5 << 20) == -1                           # no bias
    ok = {"stats": 6 << 20, "grad_weight": 7 << 20, "workspace": 8 << 20}
    assert run(back, **ok, workspace_bytes=2 * 4 * 128 * 4 - 1) == -5
    assert run(back, **{**ok, "workspace": None}, workspace_bytes=1 << 20) == -5
    assert run(back, stats=6 << 20, grad_input=2 << 20) == -2           # over the residual


@pytest.mark.gpu
@pytest.mark.parametrize("H,dtype", [(6140, "fp32"), (6136, "bf16"), (6144, "bf16"), (5640, "fp16"),
                                     (12280, "fp32"), (768, "bf16")])
def test_parameters_that_just_fill_shared_memory(H, dtype):
    """Rows whose parameters take close to 48 KB of a block's shared memory, beside its own arrays."""
    _check_all(*_inputs(450, H, DT[dtype], True, True, True), 1e-5)


# rows off the 16-byte boundary in tensors on it: every place of a first column in its 16 bytes, rows shorter
# than 16 bytes, a warp's and a block's rows, more rows than blocks, the longest rows of each variant
ODD = [(3, 1), (40, 3), (9, 5), (17, 7), (8, 9), (21, 13), (2500, 31), (2399, 255), (700, 506), (601, 1021),
       (650, 2047), (601, 2046), (599, 4095), (430, 6140), (333, 7001), (300, 8191), (170, 10239),
       (160, 16369), (150, 16370), (5, 16383)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H", ODD)
def test_rows_of_any_length(T, H, dtype):
    for branch, weight, bias, f32 in ((True, True, True, False), (False, True, False, True)):
        _check_all(*_inputs(T, H, DT[dtype], branch, weight, bias, f32), 1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,H", [(1, 5), (7, 3), (900, 37), (700, 1023), (500, 3001)])
def test_rows_of_any_length_write_nothing_else(T, H, dtype):
    """hidden in place between other values, with NaN before and behind: they are neither used nor changed."""
    f, x, w, b = _inputs(T, H, DT[dtype], True, True, True)
    room = 16
    buf = torch.full((T * H + 2 * room,), float("nan"), device="cuda", dtype=x.dtype)
    mine = buf[room:-room].view(T, H)
    assert mine.data_ptr() % 16 == 0
    mine.copy_(x)
    h_ref, y_ref = fb.layer_norm(f, x, weight=w, bias=b)
    h, y = fb.layer_norm(f, mine, weight=w, bias=b, output=mine)
    assert h is mine and torch.equal(h, h_ref) and torch.equal(y, y_ref)
    assert bool(torch.isnan(buf[:room]).all()) and bool(torch.isnan(buf[-room:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("H", [37, 1023, 3001])
def test_a_bad_row_of_any_length_stays_in_its_row(H):
    """Neighbouring rows share 16 bytes: infinities and NaN at a row's ends reach no other row, forward or
    backward (but the sums over rows)."""
    f, x, w, b = _inputs(900, H, torch.bfloat16, True, True, True)
    clean = x.clone()
    x[400, 0], x[400, -1], x[402, -1], x[404, 0] = float("inf"), float("nan"), float("inf"), float("nan")
    dy = torch.randn_like(x)
    dy[410, 0] = dy[410, -1] = float("nan")
    good = torch.ones(900, dtype=torch.bool, device="cuda")
    good[[400, 402, 404]] = False
    out = []
    for t in (x, clean):
        t = t.clone().requires_grad_()
        h, y = fb.layer_norm(f, t, weight=w, bias=b)
        out.append((h.detach(), y.detach(), torch.autograd.grad(y, t, dy)[0]))
    for got, ref in zip(*out):
        assert torch.equal(got[good].nan_to_num(7.0), ref[good].nan_to_num(7.0))
    assert bool(torch.isfinite(out[0][2][[399, 401, 403, 405, 409, 411]][:, 1:-1]).any())
    good[410] = False
    assert bool(torch.isfinite(out[0][2][good]).all())
