"""The norms before and after a block, with gate and residual scale, against 64-bit forms."""
import ctypes

import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from tests import layer_refs as R

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _inputs(T, H, dt, post, gate, pre, branch=True, seed=0, param=None):
    g = torch.Generator().manual_seed(seed + T + H)
    param = param or dt
    f = torch.randn(T, H, generator=g).to(dt).cuda() if branch else None
    big = 1 + 30.0 * (torch.rand(H, generator=g) < 0.01)
    x = (2 * big * torch.randn(T, H, generator=g)).to(dt).cuda()
    wp = (1 + 0.2 * torch.randn(H, generator=g)).to(param).cuda() if post else None
    shape = {"token": (T, 1), "channel": (H,), "full": (T, H)}.get(gate)
    gt = torch.randn(*shape, generator=g).to(param).cuda() if shape else None
    wq = (1 + 0.2 * torch.randn(H, generator=g)).to(param).cuda() if pre else None
    return f, x, wp, gt, wq


def _call(t, s, **kw):
    return fb.block_norm(t[0], t[1], post_weight=t[2], gate=t[3], pre_weight=t[4],
                         residual_scale=s, eps=EPS, **kw)


# T, H, dtype, post, gate, scale, pre, fp32 parameters
CASES = [
    (1, 1, "fp32", True, "full", 1.0, True, False),
    (1, 7168, "bf16", True, "none", 1.0, True, False),
    (3, 64, "fp16", True, "token", 0.5, True, True),
    (5, 1407, "bf16", True, "channel", 1.25, True, False),
    (7, 513, "fp32", False, "full", -0.5, True, False),
    (2, 16384, "bf16", True, "channel", 1.0, True, True),
    (2, 16384, "fp32", True, "full", 1.0, True, False),
    (2, 16383, "fp16", True, "token", 1.0, True, False),
    (17, 2048, "fp16", True, "full", 1.0, False, False),
    (301, 256, "bf16", True, "token", 0.0, True, False),
    (40, 8, "bf16", False, "none", 1.0, True, True),
    (600, 136, "fp32", True, "channel", 1.0, True, False),
    (9, 4100, "bf16", False, "channel", 2.0, True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,dtype,post,gate,s,pre,f32", CASES)
def test_forward_and_gradients(T, H, dtype, post, gate, s, pre, f32):
    dt = DT[dtype]
    t = _inputs(T, H, dt, post, gate, pre, param=torch.float32 if f32 else None)
    hidden, normed = _call(t, s)
    leaves = R.norm_leaves(*t)
    rh, ry = R.block_norm(*leaves, s, EPS)
    eh, ey, *_ = R.block_norm_bounds(*[None if v is None else v.detach() for v in leaves], s, EPS)
    R.check(hidden, rh.detach(), eh, "hidden")
    assert (normed is None) == (not pre)
    if pre:
        R.check(normed, ry.detach(), ey, "normed")

    t = [None if v is None else v.requires_grad_() for v in t]
    g = torch.Generator().manual_seed(5)
    da = torch.randn(T, H, generator=g).to(dt).cuda()
    dy = torch.randn(T, H, generator=g).to(dt).cuda() if pre else None
    h2, y2 = _call(t, s)
    assert torch.equal(h2, hidden) and (not pre or torch.equal(y2, normed))
    names = [n for n, v in zip(("branch", "residual", "post_w", "gate", "pre_w"), t)
             if v is not None]
    live = [v for v in t if v is not None]
    for a, b in ((da, dy), (None, dy), (da, None)):
        outs = [(o, r, d) for o, r, d in ((h2, rh, a), (y2, ry, b)) if d is not None]
        if not outs:
            continue
        got = torch.autograd.grad([o for o, _, _ in outs], live, [d for _, _, d in outs],
                                  retain_graph=True, allow_unused=True)
        ref = torch.autograd.grad([r for _, r, _ in outs], [v for v in leaves if v is not None],
                                  [d.double() for _, _, d in outs], retain_graph=True,
                                  allow_unused=True)
        err = R.block_norm_grad_bounds(leaves, s, EPS, a, b)
        for n, v, w, leaf in zip(names, got, ref, live):
            w = torch.zeros_like(leaf, dtype=torch.float64) if w is None else w
            assert v.dtype == leaf.dtype
            R.check(v, w, err[n], n)


def _shifted(v):
    """The same values in a tensor that starts one element off a 16-byte boundary."""
    if v is None:
        return None
    out = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape)
    return out.copy_(v)


# T, H, dtype, off the boundary: rows that take the kernels without a ring, and beside them rows
# that take the ring
@pytest.mark.gpu
@pytest.mark.parametrize("T,H,dtype,off", [(5, 200, "bf16", True), (3, 1000, "fp16", True),
                                           (2, 2500, "fp32", True), (2, 16384, "fp32", False),
                                           (6, 512, "bf16", False), (6, 513, "bf16", False)])
@pytest.mark.parametrize("branch,post,gate,pre", [(False, False, "none", True),
                                                  (True, False, "none", True),
                                                  (True, True, "none", False),
                                                  (True, True, "token", True),
                                                  (True, False, "channel", True),
                                                  (True, True, "full", True),
                                                  (True, False, "full", False)])
def test_every_form_on_every_path(T, H, dtype, off, branch, post, gate, pre):
    dt, s = DT[dtype], 0.75
    t = _inputs(T, H, dt, post, gate, pre, branch=branch)
    leaves = R.norm_leaves(*t)
    rh, ry = R.block_norm(*leaves, s, EPS)
    eh, ey, *_ = R.block_norm_bounds(*[None if v is None else v.detach() for v in leaves], s, EPS)
    if off:
        t = [_shifted(v) for v in t]
    t = [None if v is None else v.requires_grad_() for v in t]
    hidden, normed = _call(t, s)
    R.check(hidden, rh.detach(), eh, "hidden")
    if pre:
        R.check(normed, ry.detach(), ey, "normed")
    g = torch.Generator().manual_seed(5)
    da = torch.randn(T, H, generator=g).to(dt).cuda()
    dy = torch.randn(T, H, generator=g).to(dt).cuda() if pre else None
    names = [n for n, v in zip(("branch", "residual", "post_w", "gate", "pre_w"), t)
             if v is not None]
    live = [v for v in t if v is not None]
    got = torch.autograd.grad((hidden, normed) if pre else (hidden,), live, (da, dy) if pre else (da,))
    ref = torch.autograd.grad((rh, ry) if pre else (rh,), [v for v in leaves if v is not None],
                              (da.double(), dy.double()) if pre else (da.double(),))
    err = R.block_norm_grad_bounds(leaves, s, EPS, da, dy)
    for n, v, w in zip(names, got, ref):
        R.check(v, w, err[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [False, True])
def test_gradients_of_tiny_rows_without_eps(off):
    """Rows of 1e-15 with eps 0: their norms' cubes leave fp32, the gradients do not."""
    T, H, eps = 3, 264, 0.0
    g = torch.Generator().manual_seed(4)
    t = [(1e-15 * torch.randn(T, H, generator=g)).cuda(), (1e-15 * torch.randn(T, H, generator=g)).cuda(),
         (1 + torch.rand(H, generator=g)).cuda(), None, (1 + torch.rand(H, generator=g)).cuda()]
    t[2] = t[2] * 1e-15                      # the normed branch is of the residual's size
    da = (1e15 * torch.randn(T, H, generator=g)).cuda()
    dy = torch.randn(T, H, generator=g).cuda()
    leaves = R.norm_leaves(*t)
    rh, ry = R.block_norm(*leaves, 1.0, eps)
    names = ("branch", "residual", "post_w", "pre_w")
    ref = torch.autograd.grad((rh, ry), [v for v in leaves if v is not None],
                              (da.double(), dy.double()))
    err = R.block_norm_grad_bounds(leaves, 1.0, eps, da, dy)
    t = [None if v is None else (_shifted(v) if off else v).requires_grad_() for v in t]
    h, y = fb.block_norm(t[0], t[1], post_weight=t[2], pre_weight=t[4], eps=eps)
    got = torch.autograd.grad((h, y), [v for v in t if v is not None], (da, dy))
    for n, v, w in zip(names, got, ref):
        R.check(v, w, err[n], n)


@pytest.mark.gpu
def test_gradients_against_differences():
    """<gradient, v> against central differences of the 64-bit form along random v."""
    s, T, H = 0.7, 6, 72
    t = _inputs(T, H, torch.float32, True, "channel", True)
    t = [v.requires_grad_() for v in t]
    g = torch.Generator().manual_seed(8)
    da, dy = (torch.randn(T, H, generator=g).cuda() for _ in range(2))
    got = torch.autograd.grad(_call(t, s), t, (da, dy))
    base = [v.detach().double() for v in t]
    err = R.block_norm_grad_bounds(base, s, EPS, da, dy)

    def loss(v):
        h, y = R.block_norm(*v, s, EPS)
        return float((h * da.double()).sum() + (y * dy.double()).sum())
    step = 1e-5
    for i, n in enumerate(("branch", "residual", "post_w", "gate", "pre_w")):
        v = torch.randn(base[i].shape, generator=g).double().cuda()
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + step * v, base[i] - step * v
        num = (loss(hi) - loss(lo)) / (2 * step)
        mine = float((got[i].double() * v).sum())
        # the gradient's own bound, and 1e-7 of the terms for the differences (step^2 and 1e-16/step)
        room = float((R.tol(got[i].double(), err[n], torch.float32) * v.abs()).sum())
        assert abs(mine - num) <= room + 1e-7 * float((got[i].double() * v).abs().sum()), n


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,dtype", [(1, 128, "bf16"), (16, 7168, "bf16"), (5, 1280, "fp16"),
                                       (3, 384, "fp32"), (2, 16384, "fp32")])
def test_quantised_output(T, H, dtype):
    t = _inputs(T, H, DT[dtype], True, "token", True)
    t[1][0, :128] = 0
    t[0][0, :128] = 0                          # a block of zeros: the smallest scale
    hidden, (q, scale) = _call(t, 1.0, quantize=True)
    v = [None if x is None else x.double() for x in t]
    rh, ry = R.block_norm(*v, 1.0, EPS)
    eh, ey, *_ = R.block_norm_bounds(*v, 1.0, EPS)
    R.check(hidden, rh, eh, "hidden")
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (H // 128, T)
    amax = ry.view(T, H // 128, 128).abs().amax(2).clamp(min=1e-30)
    e_blk = ey.view(T, H // 128, 128).amax(2)
    # the maximum's error over 448, one division's rounding and 1e-30's own
    assert bool(((scale.t().double() - amax / 448).abs()
                 <= e_blk / 448 + 2 * R.U * amax / 448).all())
    # half an e4m3 step of the value, half the smallest step (2^-10) of the scale, and y's error
    back = q.double() * scale.t().double().repeat_interleave(128, 1)
    room = ey * 1.1 + 2.0 ** -4 * ry.abs() * (1 + 1e-5) \
        + 2.0 ** -10 * scale.t().double().repeat_interleave(128, 1)
    assert bool(((back - ry).abs() <= room).all())


@pytest.mark.gpu
def test_quantised_output_is_the_expert_layers_input():
    """The e4m3 form against quantising the fp32 form's values by the layer's convention, bit for
    bit. Both in fp32: a bf16 row is summed in another order (groups of eight, not four), which may
    move the norm's factor by a rounding."""
    x = torch.randn(24, 7168, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()
    x = x.float()
    w = torch.ones(7168, device="cuda")
    h, (q, s) = fb.block_norm(None, x, pre_weight=w, quantize=True)
    assert h is x
    _, y = fb.block_norm(None, x, pre_weight=w)
    blocks = y.view(24, 56, 128)
    scale = blocks.abs().amax(2).clamp(min=1e-30) / torch.full((24, 56), 448.0, device="cuda")
    assert torch.equal(s.t(), scale)
    want = (blocks / scale[:, :, None]).to(torch.float8_e4m3fn).view(24, 7168)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.gpu
def test_in_place_and_off_the_16_byte_boundary():
    t = _inputs(33, 256, torch.bfloat16, True, "token", True)
    hidden, normed = _call(t, 0.5)
    res = t[1].clone()
    h2, y2 = _call((t[0], res, *t[2:]), 0.5, output=res)
    assert h2 is res and torch.equal(res, hidden) and torch.equal(y2, normed)
    flat = torch.empty(33 * 256 + 1, dtype=torch.bfloat16, device="cuda")
    off = flat[1:].view(33, 256)
    off.copy_(t[1])
    h3, y3 = _call((t[0], off, *t[2:]), 0.5)
    v = [x.double() for x in t]
    eh, ey, *_ = R.block_norm_bounds(*v, 0.5, EPS)
    rh, ry = R.block_norm(*v, 0.5, EPS)
    R.check(h3, rh, eh, "hidden")
    R.check(y3, ry, ey, "normed")
    with pytest.raises(RuntimeError, match="ALIGN"):
        _call((t[0], off, *t[2:]), 0.5, quantize=True)


@pytest.mark.gpu
def test_zero_rows_and_non_finite_rows_stay_in_their_row():
    t = _inputs(4, 64, torch.bfloat16, True, "none", True)
    t[0][1], t[1][1] = 0, 0
    t[0][2, 3] = float("inf")
    t[1][3, 5] = float("nan")
    h, y = _call(t, 1.0)
    assert bool(torch.isfinite(h[0]).all()) and not bool(h[1].any()) and not bool(y[1].any())
    assert bool(torch.isnan(h[2]).any()) and bool(torch.isnan(y[3]).all())
    for v in (t[0], t[1], t[2], t[4]):
        v.requires_grad_()
    h, y = _call(t, 1.0)
    df, dx = torch.autograd.grad(y[:2].float().sum(), (t[0], t[1]))
    # a row of zeros: 1/sqrt(eps) is finite, and so are its gradients
    assert bool(torch.isfinite(df[:2]).all()) and bool(torch.isfinite(dx[:2]).all())


@pytest.mark.gpu
def test_no_tokens():
    t = [v.requires_grad_() for v in _inputs(0, 64, torch.bfloat16, True, "channel", True)]
    h, y = _call(t, 1.0)
    grads = torch.autograd.grad((h.sum() + y.sum()), t)
    assert h.shape == y.shape == (0, 64) and all(not bool(v.any()) for v in grads)


@pytest.mark.gpu
def test_expanded_gradients_and_a_captured_training_step():
    """A gradient that autograd hands over as an expanded scalar, and the same step in a graph."""
    t = [v.requires_grad_() for v in _inputs(70, 192, torch.float32, True, "channel", True)]
    g0 = torch.autograd.grad(sum(o.sum() for o in _call(t, 1.0)), t)
    da = torch.ones(70, 192, device="cuda")
    g1 = torch.autograd.grad(_call(t, 1.0), t, (da, da))
    assert all(torch.equal(a, b) for a, b in zip(g0, g1))
    del g1
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(_call(t, 1.0), t, (da, da))
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = torch.autograd.grad(_call(t, 1.0), t, (da, da))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(g0, got))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    f, x, wp, gt, wq = _inputs(4, 64, torch.bfloat16, True, "token", True)
    ok = dict(post_weight=wp, gate=gt, pre_weight=wq)
    with pytest.raises(TypeError, match="branch"):
        fb.block_norm(f.float(), x, **ok)
    with pytest.raises(ValueError, match="branch"):
        fb.block_norm(f[:3], x, **ok)
    with pytest.raises(ValueError, match="need a branch"):
        fb.block_norm(None, x, **ok)
    with pytest.raises(TypeError, match="post_weight"):
        fb.block_norm(f, x, **{**ok, "post_weight": wp.half()})
    with pytest.raises(ValueError, match="gate must have shape"):
        fb.block_norm(f, x, **{**ok, "gate": gt.view(4)})
    with pytest.raises(ValueError, match="contiguous"):
        fb.block_norm(f, x.t().contiguous().t(), **ok)
    with pytest.raises(ValueError, match="hidden size"):
        fb.block_norm(None, torch.zeros((1, 16385), device="cuda"))
    with pytest.raises(ValueError, match="multiple of 128"):
        fb.block_norm(f, x, quantize=True, **ok)
    with pytest.raises(ValueError, match="pre_weight"):
        fb.block_norm(f, x, quantize=True)
    with pytest.raises(ValueError, match="no gradient"):
        t = _inputs(2, 128, torch.bfloat16, True, "none", True)
        fb.block_norm(t[0].requires_grad_(), t[1], pre_weight=t[4], quantize=True)
    with pytest.raises(ValueError, match="gradients"):
        fb.block_norm(f.clone().requires_grad_(), x, output=x, **ok)
    with pytest.raises(RuntimeError, match="SHAPE"):
        fb.block_norm(f, x, output=f, **ok)


def test_refusals_on_the_host():
    with pytest.raises(ValueError, match="CUDA"):
        fb.block_norm(None, torch.zeros((2, 8)))
    lib = _lib.load()
    size = ctypes.c_size_t()
    assert lib.fmoe_block_norm_workspace_size(5, 64, ctypes.byref(size)) == 0
    assert size.value == 3 * 5 * 64 * 4
    assert lib.fmoe_block_norm_workspace_size(5, 16385, ctypes.byref(size)) == -2
    assert lib.fmoe_block_norm_workspace_size(5, 64, None) == -1
    assert lib.fmoe_block_norm(None, None) == -1
    a = _lib.FmoeBlockNormArgs()

    def run(fn=lib.fmoe_block_norm, **kw):
        for k in ("hidden", "normed", "normed_q", "normed_scale", "stats", "grad_hidden",
                  "grad_normed", "grad_branch", "grad_residual", "grad_post_weight", "grad_gate",
                  "grad_pre_weight", "workspace"):
            setattr(a, k, None)
        a.workspace_bytes = 0
        a.num_tokens, a.hidden_size, a.dtype, a.gate_kind = 4, 128, 1, 0
        a.branch, a.residual, a.post_weight, a.gate, a.pre_weight = 1 << 20, 2 << 20, 3 << 20, 0, 0
        a.post_weight_dtype = a.gate_dtype = a.pre_weight_dtype = 1
        for k, v in kw.items():
            setattr(a, k, v)
        return fn(ctypes.byref(a), None)
    assert run(hidden_size=0) == -2 and run(hidden_size=16385) == -2 and run(num_tokens=-1) == -2
    assert run(gate_kind=4) == -2 and run(dtype=5) == -6 and run(post_weight_dtype=2) == -6
    assert run(residual=None) == -1 and run(branch=None) == -1 and run(gate_kind=1) == -1
    assert run(normed=4 << 20) == -1                         # normed without pre_weight
    assert run(pre_weight=5 << 20) == -1                     # and the other way round
    assert run(residual=(2 << 20) + 1) == -3
    assert run(hidden=(1 << 20) + 64) == -2                  # over the branch
    q = dict(pre_weight=5 << 20, normed_q=6 << 20, normed_scale=7 << 20)
    assert run(hidden_size=136, **q) == -2 and run(residual=(2 << 20) + 8, **q) == -3
    assert run(**{**q, "normed_scale": None}) == -1
    assert run(num_tokens=0) == 0 and run() == 0             # nothing asked for
    back = lib.fmoe_block_norm_backward
    assert run(back, grad_residual=6 << 20) == -1            # no stats
    assert run(back, grad_post_weight=6 << 20, stats=8 << 20) == -5
    assert run(back, grad_gate=6 << 20, stats=8 << 20) == -1
    assert run(back, grad_residual=2 << 20, stats=8 << 20) == -2


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    t = [v.requires_grad_() for v in _inputs(3, 32, torch.float32, True, "none", True)
         if v is not None]
    h, _ = fb.block_norm(t[0], t[1], post_weight=t[2], pre_weight=t[3])
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(h.sum(), t[0], create_graph=True)
