"""Int8 quantisation and products, dense and per expert, against exact integer arithmetic."""
import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from tests import layer_refs as R

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int8(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K", [(1, 1), (3, 16), (5, 33), (1, 7168), (257, 2047), (64, 4104),
                                 (2, 20000), (1000, 128), (3, 2056)])
def test_quantize(T, K, dtype):
    g = _gen(T + K)
    x = (torch.randn(T, K, generator=g, device="cuda")
         * torch.exp(3 * torch.randn(T, 1, generator=g, device="cuda"))).to(DT[dtype])
    x[0, 0] = 0
    q, scale = fb.quantize_int8(x)
    # the row factors reach exp(9): some fp16 rows hold an infinity, which the scale carries on
    fine = torch.isfinite(x).all(1)
    assert bool((fine == torch.isfinite(scale)).all()) and not bool(q[~fine].any())
    rq, rs = R.quantize(x[fine])
    assert torch.equal(q[fine].double(), rq)
    # one fp32 division
    assert bool(((scale[fine].double() - rs).abs() <= R.U * rs).all())


@pytest.mark.gpu
def test_quantize_ties_extremes_and_non_finite():
    rows = []
    for amax in (127.0, 254.0, 3.0, 1.0, 2.0 ** -100, 2.0 ** 120, 1.5e38 * 2):
        k = torch.arange(-127, 127, dtype=torch.float64) + 0.5     # every tie
        rows.append(torch.cat([k * amax / 127, torch.tensor([amax, -amax], dtype=torch.float64)]))
    x = torch.stack(rows).to(torch.bfloat16).cuda()
    q, _ = fb.quantize_int8(x)
    assert torch.equal(q.double(), R.quantize(x)[0])
    z = torch.zeros(3, 40, dtype=torch.bfloat16, device="cuda")
    z[1] = 1e-38                                       # below the smallest scale
    z[2, 3] = -0.0
    q, s = fb.quantize_int8(z)
    assert not bool(q.any()) and bool((s > 0).all())
    bad = torch.ones(3, 64, dtype=torch.float16, device="cuda")
    bad[0, 5], bad[1, 9] = float("nan"), float("-inf")
    q, s = fb.quantize_int8(bad)
    assert not bool(torch.isfinite(s[:2]).any()) and bool(torch.isfinite(s[2]))
    w = _int8(_gen(0), 32, 64)
    y = fb.int8_matmul(q, w, s, torch.ones(32, device="cuda"))
    assert bool(torch.isnan(y[:2]).all()) and bool(torch.isfinite(y[2]).all())


# M, N, K: one token to several tiles, odd sizes, a K tail inside a 128-byte block, short K
SIZES = [(1, 1, 16), (1, 4096, 7168), (2, 128, 144), (15, 129, 128), (16, 257, 2048),
         (17, 100, 400), (64, 2047, 512), (65, 128, 1040), (130, 384, 4096), (255, 65, 272),
         (300, 1000, 1024), (517, 2047, 7168), (1025, 130, 96), (2049, 256, 2064), (33, 7168, 16),
         (1, 3, 32), (2, 17, 7168), (3, 4097, 2064), (4, 1030, 7168), (4, 33, 11776), (4, 33, 11792)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SIZES)
def test_matmul(M, N, K):
    g = _gen(M + N + K)
    a, w = _int8(g, M, K), _int8(g, N, K)
    a_s = torch.rand(M, generator=g, device="cuda") + 0.01
    w_s = torch.rand(N, generator=g, device="cuda") * 1e-3
    bias = torch.randn(N, generator=g, device="cuda") * 10
    for name, b in (("bf16", None), ("fp32", bias), ("fp16", bias * 0)):
        if name == "fp16":          # keep the products inside fp16's range
            w_s = w_s * 1e-3
        ref, err = R.product(a, w, a_s, w_s, b)
        y = fb.int8_matmul(a, w, a_s, w_s, b, out_dtype=DT[name])
        R.check(y, ref, err, name)
    assert fb.int8_status() == 0


@pytest.mark.gpu
def test_matmul_extreme_sums():
    """The largest sums: -128 * -128 and 127 * -128 over the longest K stay exact in int32."""
    K = 131056
    a = torch.full((2, K), -128, dtype=torch.int8, device="cuda")
    a[1] = 127
    w = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one = torch.ones(3, device="cuda")
    y = fb.int8_matmul(a, w, one[:2], one, out_dtype=torch.float32)
    ref = a.double() @ w.double().t()
    R.check(y, ref, R.U * ref.abs(), "sums")


# R, E, N, K, counts per expert (the rest of R lies behind the last expert)
GROUPS = [
    (1, 1, 128, 128, [1]),
    (5, 4, 130, 256, [0, 3, 0, 2]),
    (64, 32, 512, 1024, None),
    (100, 8, 96, 144, [0, 0, 50, 1, 0, 17, 0, 0]),       # a tail of 32 rows
    (1000, 5, 300, 512, [257, 0, 600, 16, 127]),
    (700, 256, 64, 128, None),
    (40, 3, 200, 4096, [0, 0, 0]),                       # no live row at all
    (3000, 2, 128, 2064, [2999, 1]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("Rn,E,N,K,counts", GROUPS)
def test_expert_matmul(Rn, E, N, K, counts):
    g = _gen(Rn + E)
    if counts is None:
        p = torch.rand(E, generator=g, device="cuda") ** 2
        ids = torch.multinomial(p, Rn, replacement=True, generator=g)
        counts = torch.bincount(ids, minlength=E).tolist()
    base = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    live = int(base[-1])
    rows, w = _int8(g, Rn, K), _int8(g, E, N, K)
    r_s = torch.rand(Rn, generator=g, device="cuda") + 0.01
    w_s = torch.rand(E, N, generator=g, device="cuda") * 1e-3
    ref = torch.zeros(Rn, N, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(ref)
    for e in range(E):
        lo, hi = int(base[e]), int(base[e + 1])
        ref[lo:hi], err[lo:hi] = R.product(rows[lo:hi], w[e], r_s[lo:hi], w_s[e])
    y = fb.int8_expert_matmul(rows, w, r_s, w_s, base.cuda())
    R.check(y, ref, err, "rows")
    out = torch.full((Rn, N), 3.0, device="cuda")
    fb.int8_expert_matmul(rows, w, r_s, w_s, base.cuda(), output=out)
    ref[live:] = 3.0
    R.check(out, ref, err, "given output")
    assert fb.int8_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("Rn,N,lo,hi", [(9, 33, 4, 6), (40, 64, 40, 40), (700, 2047, 300, 311),
                                        (2000, 130, 1, 1999), (3, 1, 1, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_no_expert(Rn, N, lo, hi, dtype):
    """A part of an order's experts: rows before the first and behind the last are zero in a new
    tensor and stay in a given one, at every alignment of their ends."""
    g = _gen(Rn)
    base = torch.tensor([lo, (lo + hi) // 2, hi], dtype=torch.int32, device="cuda")
    rows, w = _int8(g, Rn, 48), _int8(g, 2, N, 48)
    one, ws = torch.ones(Rn, device="cuda"), torch.ones(2, N, device="cuda")
    mid = (lo + hi) // 2
    ref = torch.zeros(Rn, N, dtype=torch.float64, device="cuda")
    ref[lo:mid] = rows[lo:mid].double() @ w[0].double().t()
    ref[mid:hi] = rows[mid:hi].double() @ w[1].double().t()
    # dirty blocks of the allocator's, so that a row that is not written shows
    dirt = [torch.full((Rn, N), 5.0, dtype=dtype, device="cuda") for _ in range(3)]
    del dirt
    y = fb.int8_expert_matmul(rows, w, one, ws, base, out_dtype=dtype)
    assert torch.equal(y, ref.to(dtype))
    flat = torch.full((Rn * N + 1,), 3.0, dtype=dtype, device="cuda")
    out = flat[1:].view(Rn, N)
    fb.int8_expert_matmul(rows, w, one, ws, base, output=out)
    ref[:lo], ref[hi:] = 3.0, 3.0
    assert torch.equal(out, ref.to(dtype)) and float(flat[0]) == 3.0


@pytest.mark.gpu
def test_expert_bases_out_of_range_are_clamped():
    """Bases below 0, above R or stepping back stay inside the tensors."""
    g = _gen(9)
    rows, w = _int8(g, 20, 64), _int8(g, 3, 48, 64)
    one = torch.ones(20, device="cuda")
    ws = torch.ones(3, 48, device="cuda")
    base = torch.tensor([-7, 8, 8, 1000], dtype=torch.int32, device="cuda")
    y = fb.int8_expert_matmul(rows, w, one, ws, base, out_dtype=torch.float32)
    ref = torch.cat([rows[:8].double() @ w[0].double().t(), rows[8:].double() @ w[2].double().t()])
    assert torch.equal(y.double(), ref)
    back = torch.tensor([0, 12, 5, 20], dtype=torch.int32, device="cuda")
    y = fb.int8_expert_matmul(rows, w, one, ws, back, out_dtype=torch.float32)
    assert torch.equal(y[:5].double(), rows[:5].double() @ w[0].double().t())
    assert torch.equal(y[12:].double(), rows[12:].double() @ w[2].double().t())


@pytest.mark.gpu
def test_same_bits_again_and_in_two_graphs_at_once():
    """Two captured graphs replayed side by side on two streams give what eager calls give."""
    g = _gen(3)
    sets = []
    for M, N, K in ((1, 1024, 7168), (300, 512, 2048)):
        x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
        w = _int8(g, N, K)
        w_s = torch.rand(N, generator=g, device="cuda")

        def step(x=x, w=w, w_s=w_s):
            q, s = fb.quantize_int8(x)
            return fb.int8_matmul(q, w, s, w_s)
        want = step()
        assert torch.equal(want, step())
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
        sets.append((graph, stream, got, want, step))    # step holds the graph's inputs
    for _ in range(20):
        for graph, stream, *_ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _ in sets:
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_empty_calls_and_refusals_on_the_gpu():
    a = torch.zeros((4, 32), dtype=torch.int8, device="cuda")
    w = torch.zeros((6, 32), dtype=torch.int8, device="cuda")
    s4, s6 = torch.ones(4, device="cuda"), torch.ones(6, device="cuda")
    assert fb.int8_matmul(a[:0], w, s4[:0], s6).shape == (0, 6)
    q, s = fb.quantize_int8(torch.zeros((0, 8), device="cuda", dtype=torch.bfloat16))
    assert q.shape == (0, 8) and s.shape == (0,)
    base = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert fb.int8_expert_matmul(a[:0], w[None], s4[:0], s6[None], base).shape == (0, 6)
    with pytest.raises(TypeError, match="bfloat16"):
        fb.quantize_int8(torch.zeros((2, 8), device="cuda"))
    with pytest.raises(TypeError, match="int8"):
        fb.int8_matmul(a.float(), w, s4, s6)
    with pytest.raises(ValueError, match="fit"):
        fb.int8_matmul(a, w[:, :16].contiguous(), s4, s6)
    with pytest.raises(ValueError, match="multiple of 16"):
        fb.int8_matmul(a[:, :24].contiguous(), w[:, :24].contiguous(), s4, s6)
    with pytest.raises(ValueError, match="contiguous"):
        fb.int8_matmul(a, torch.zeros((32, 6), dtype=torch.int8, device="cuda").t(), s4, s6)
    with pytest.raises(ValueError, match="a_scale"):
        fb.int8_matmul(a, w, s6, s6)
    with pytest.raises(TypeError, match="b_scale"):
        fb.int8_matmul(a, w, s4, s6.double())
    with pytest.raises(ValueError, match="bias"):
        fb.int8_matmul(a, w, s4, s6, s4)
    with pytest.raises(TypeError, match="out_dtype"):
        fb.int8_matmul(a, w, s4, s6, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="output"):
        fb.int8_matmul(a, w, s4, s6, output=torch.zeros((4, 5), device="cuda"))
    with pytest.raises(ValueError, match="expert_base"):
        fb.int8_expert_matmul(a, w[None], s4, s6[None], base[:1])
    with pytest.raises(RuntimeError, match="ALIGN"):
        flat = torch.zeros(4 * 32 + 1, dtype=torch.int8, device="cuda")
        fb.int8_matmul(flat[1:].view(4, 32), w, s4, s6)


def test_refusals_on_the_host():
    with pytest.raises(ValueError, match="CUDA"):
        fb.quantize_int8(torch.zeros((2, 8), dtype=torch.bfloat16))
    lib = _lib.load()
    f = lib.fmoe_int8_matmul
    A, B, S, W, O = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
    assert f(A, B, S, W, None, 4, 8, 24, O, 1, None) == -2       # K not a multiple of 16
    assert f(A, B, S, W, None, 4, 8, 131072, O, 1, None) == -2   # sums could leave int32
    assert f(A, B, S, W, None, 4, 0, 32, O, 1, None) == -2
    assert f(A, B, S, W, None, -1, 8, 32, O, 1, None) == -2
    assert f(A, B, S, W, None, 4, 8, 32, O, 9, None) == -6
    assert f(A, B, S, W, None, 0, 8, 32, O, 1, None) == 0
    assert f(A, None, S, W, None, 4, 8, 32, O, 1, None) == -1
    assert f(A + 8, B, S, W, None, 4, 8, 32, O, 1, None) == -3
    assert f(A, B, S, W, None, 4, 8, 32, O + 1, 1, None) == -3
    assert f(A, B, S, W, None, 4, 8, 32, A + 64, 1, None) == -2  # output over its input
    e = lib.fmoe_int8_expert_matmul
    assert e(A, B, S, W, None, 4, 2, 8, 32, O, 1, 1, None) == -1
    assert e(A, B, S, W, 64, 4, 257, 8, 32, O, 1, 1, None) == -2
    assert e(A, B, S, W, 64, 4, 256, 2 ** 24, 32, O, 1, 1, None) == -2
    assert lib.fmoe_quantize_int8(A, 0, 4, 8, B, S, None) == -6  # fp32 input
    assert lib.fmoe_quantize_int8(A, 1, 4, 0, B, S, None) == -2
    assert lib.fmoe_quantize_int8(A, 1, 4, 8, A, S, None) == -2
    assert lib.fmoe_quantize_int8(A, 1, 0, 8, None, None, None) == 0
    assert lib.fmoe_int8_status(None, None) == -1
    assert lib.fmoe_debug_arm_int8_timeout(10) == -2             # below 100 us
    assert lib.fmoe_debug_arm_int8_timeout(3_000_000_000) == -2  # above 2 s


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(40, 1024, 4096), (200, 12800, 256), (600, 2048, 4096),
                                   (2048, 4096, 256)])
def test_a_wait_that_runs_out_ends_the_product(M, N, K):
    """One CTA per tile, its K split, CTA pairs and theirs: a wait that nothing ends gives up after
    its 5 ms, the status says so once, and the next product (which needs the same tensor memory) is
    right."""
    import time
    g = _gen(M)
    a, w = _int8(g, M, K), _int8(g, N, K)
    a_s, w_s = torch.rand(M, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    fb.int8_matmul(a, w, a_s, w_s)
    assert fb.int8_status() == 0
    assert _lib.load().fmoe_debug_arm_int8_timeout(5_000_000) == 0
    t0 = time.perf_counter()
    fb.int8_matmul(a, w, a_s, w_s)
    assert fb.int8_status() == _lib.STATUS_TIMEOUT_INT8
    assert time.perf_counter() - t0 < 1.0
    assert fb.int8_status() == 0
    y = fb.int8_matmul(a, w, a_s, w_s)
    ref, err = R.product(a, w, a_s, w_s)
    R.check(y, ref, err, "after")
    assert fb.int8_status() == 0
