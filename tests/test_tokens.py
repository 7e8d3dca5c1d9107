"""Tokens sorted by expert and back, and the gradients, against plain 64-bit forms."""
import ctypes

import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from flashinfer_b200.tokens import ExpertOrder
from tests import layer_refs as R
from tests.layer_refs import U

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ids(T, K, E, lo, hi, seed, repeat=False):
    """int32 picks in [lo, hi); with ``repeat`` a token may pick an expert twice."""
    g = torch.Generator().manual_seed(seed)
    if repeat or hi - lo < K:
        return torch.randint(lo, hi, (T, K), generator=g, dtype=torch.int32)
    return (torch.rand(T, hi - lo, generator=g).topk(K, 1).indices + lo).to(torch.int32)


# T, K, local experts, offset, ids from, to, align
ORDERS = [
    (1, 1, 1, 0, 0, 1, 1),
    (1, 8, 256, 0, 0, 256, 1),
    (3, 8, 32, 64, 0, 256, 16),
    (7, 5, 8, 0, -1, 9, 128),          # ids without an expert on both sides
    (33, 3, 20, 40, 100, 160, 1),      # nothing local
    (511, 8, 256, 0, 0, 256, 1),       # one block
    (513, 8, 256, 0, 0, 256, 1),       # two passes over several blocks
    (1237, 6, 20, 40, 0, 160, 16),
    (4099, 2, 1024, 0, 0, 1024, 3),
    (2500, 8, 3, 0, 0, 3, 1),          # every pick several times in a token
    (513, 8, 257, 0, 0, 512, 1),       # too many experts for one cluster
    (8191, 8, 200, 20, -1, 256, 7),    # the most picks of one cluster, nearly
    (8193, 8, 256, 0, 0, 256, 1),      # one token more than a cluster takes
    (20000, 8, 256, 0, 0, 256, 128),   # blocks of more than the least chunk
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,E,lo,a,b,align", ORDERS)
def test_order_tables(T, K, E, lo, a, b, align):
    ids = _ids(T, K, E, a, b, T + K, repeat=K > b - a)
    base, row_pick, pick_row = R.order(ids, lo, E, align)
    o = fb.sort_by_expert(ids.cuda(), E, lo, align=align)
    assert o.expert_base.tolist() == base
    assert o.row_pick.tolist() == row_pick
    assert torch.equal(o.pick_row.cpu(), pick_row)
    again = fb.sort_by_expert(ids.cuda(), E, lo, align=align)
    assert torch.equal(again.row_pick, o.row_pick)


@pytest.mark.gpu
def test_order_of_extreme_ids_and_no_tokens():
    ids = torch.tensor([[2 ** 31 - 1, -2 ** 31, 5]], dtype=torch.int32, device="cuda")
    o = fb.sort_by_expert(ids, 4, 3)
    assert o.expert_base.tolist() == [0, 0, 0, 1, 1]
    assert o.row_pick.tolist() == [2, -1, -1] and o.pick_row.tolist() == [[-1, -1, 0]]
    o = fb.sort_by_expert(torch.empty((0, 8), dtype=torch.int32, device="cuda"), 4)
    assert o.expert_base.tolist() == [0] * 5 and o.num_rows == 0
    x = torch.empty((0, 16), device="cuda", requires_grad=True)
    rows = fb.sort_tokens(x, o)
    y = fb.unsort_tokens(rows, o, torch.empty((0, 8), device="cuda"))
    assert rows.shape == (0, 16) and y.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 16)


# T, K, E, offset, ids from, to, align, H
ROWS = [
    (1, 8, 256, 0, 0, 256, 1, 7168),
    (5, 8, 8, 4, -2, 16, 16, 24),
    (37, 2, 4, 0, 0, 4, 1, 1),
    (64, 9, 16, 0, 0, 16, 1, 1407),    # more than eight picks, odd rows
    (67, 3, 7, 1, 0, 9, 4, 2047),      # odd rows of several blocks, some picks not local
    (13, 2, 3, 0, 0, 3, 1, 8209),
    (130, 6, 20, 40, 0, 160, 128, 514),
    (700, 8, 32, 0, 0, 256, 1, 256),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,K,E,lo,a,b,align,H", ROWS)
def test_sort_unsort_and_gradients(T, K, E, lo, a, b, align, H, dtype):
    g = torch.Generator().manual_seed(T * 31 + H)
    dt = DT[dtype]
    ids = _ids(T, K, E, a, b, T)
    _, row_pick, pick_row = R.order(ids, lo, E, align)
    o = fb.sort_by_expert(ids.cuda(), E, lo, align=align)
    n = o.num_rows
    pick_row = pick_row.cuda()
    x = torch.randn(T, H, generator=g).to(dt).cuda().requires_grad_()
    out = torch.randn(n, H, generator=g).to(dt).cuda()
    none = torch.tensor(row_pick, device="cuda") < 0
    out[none] = float("nan")                     # rows without a pick are not read
    out.requires_grad_()
    w = torch.randn(T, K, generator=g).cuda()
    w[pick_row < 0] = float("inf")               # nor are the weights of picks without a row
    w.requires_grad_()
    g_rows = torch.randn(n, H, generator=g).to(dt).cuda()
    g_rows[none] = float("nan")
    g_y = torch.randn(T, H, generator=g).to(dt).cuda()

    rows = fb.sort_tokens(x, o)
    assert torch.equal(rows.double(), R.rows_of(x, row_pick, K))
    y = fb.unsort_tokens(out, o, w)
    ref, mag = R.unsort(out.detach(), pick_row, w.detach())
    R.check(y.detach(), ref, K * U * mag, "y")
    dx, dout, dw = torch.autograd.grad((rows, y), (x, out, w), (g_rows, g_y))
    ref, mag = R.unsort(g_rows, pick_row, None)
    R.check(dx, ref, K * U * mag, "dx")
    w_row = torch.zeros(n, dtype=torch.float64, device="cuda")
    w_row[~none] = w.detach().double().view(-1)[torch.tensor(row_pick, device="cuda")[~none]]
    ref = w_row[:, None] * R.rows_of(g_y, row_pick, K)
    R.check(dout, ref, U * ref.abs(), "d rows")
    has = pick_row >= 0
    terms = g_y.double()[:, None, :] * torch.where(
        has[:, :, None], out.detach().double()[pick_row.clamp(min=0).long()], 0.0)
    R.check(dw, terms.sum(2), H * U * terms.abs().sum(2), "dw")
    # without weights: ones; the weights' gradient is not asked for
    plain = fb.unsort_tokens(out, o)
    ref, mag = R.unsort(out.detach(), pick_row, None)
    R.check(plain.detach(), ref, K * U * mag, "y without weights")
    (dplain,) = torch.autograd.grad(plain, out, g_y)
    assert torch.equal(dplain.double(), R.rows_of(g_y, row_pick, K))


@pytest.mark.gpu
def test_gradients_against_differences():
    """<gradient, v> against central differences of the 64-bit form along random v."""
    T, K, E, H = 9, 3, 5, 40
    ids = _ids(T, K, E, -1, E + 1, 3, repeat=True)
    _, row_pick, pick_row = R.order(ids, 0, E, 4)
    o = fb.sort_by_expert(ids.cuda(), E, align=4)
    pick_row = pick_row.cuda()
    g = torch.Generator().manual_seed(1)
    rows, w, g_y, v_r, v_w = (torch.randn(*s, generator=g).cuda() for s in (
        (o.num_rows, H), (T, K), (T, H), (o.num_rows, H), (T, K)))
    rows.requires_grad_()
    w.requires_grad_()
    d_r, d_w = torch.autograd.grad(fb.unsort_tokens(rows, o, w), (rows, w), g_y)

    def loss(r, ww):
        return float((R.unsort(r, pick_row, ww)[0] * g_y.double()).sum())
    h = 1e-4
    r64, w64 = rows.detach().double(), w.detach().double()
    # the loss is linear in each argument: differences are exact up to float64 rounding
    for d, v, lo, hi in ((d_r, v_r, (r64 - h * v_r, w64), (r64 + h * v_r, w64)),
                         (d_w, v_w, (r64, w64 - h * v_w), (r64, w64 + h * v_w))):
        num = (loss(*hi) - loss(*lo)) / (2 * h)
        got = float((d.double() * v.double()).sum())
        assert abs(got - num) <= 1e-6 * float((d.double() * v.double()).abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H", [(torch.int8, 7168), (torch.int8, 33), (torch.uint8, 1),
                                     (torch.int8, 1001), (torch.uint8, 5003),
                                     (torch.float8_e4m3fn, 130), (torch.float32, 0),
                                     (torch.int64, 3)])
def test_sort_any_element_type(dtype, H):
    T, K, E = 40, 4, 6
    ids = _ids(T, K, E, 0, 12, 5)
    _, row_pick, _ = R.order(ids, 0, E, 8)
    o = fb.sort_by_expert(ids.cuda(), E, align=8)
    shape = (T, H) if H else (T,)
    x = torch.randint(-99, 99, shape, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    rows = fb.sort_tokens(x, o)
    got = rows.view(torch.uint8) if dtype == torch.float8_e4m3fn else rows
    src = x.view(torch.uint8) if dtype == torch.float8_e4m3fn else x
    ref = R.rows_of(src.reshape(T, -1), row_pick, K)
    assert rows.dtype == dtype and rows.shape == (o.num_rows,) + shape[1:]
    assert torch.equal(got.reshape(o.num_rows, -1).double(), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("shift,H", [(0, 64), (1, 64), (0, 333), (1, 333)])
def test_given_output_keeps_the_rows_behind(shift, H):
    """Rows from expert_base[E] on stay as they were, padding rows inside are zeroed; a tensor that
    starts off a 16-byte boundary gives the same rows."""
    T, K, E = 21, 2, 3
    ids = _ids(T, K, E, 0, 6, 8)
    base, row_pick, pick_row = R.order(ids, 0, E, 16)
    o = fb.sort_by_expert(ids.cuda(), E, align=16)
    store = torch.zeros(T * H + 1, dtype=torch.bfloat16, device="cuda")
    x = store[shift:shift + T * H].view(T, H)
    x.copy_(torch.randn(T, H, generator=torch.Generator().manual_seed(0)))
    room = torch.full((o.num_rows * H + 1,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = room[shift:shift + o.num_rows * H].view(o.num_rows, H)
    assert fb.sort_tokens(x, o, output=out) is out
    ref = R.rows_of(x, row_pick, K)
    ref[base[-1]:] = 7.0
    assert torch.equal(out.double(), ref)
    assert float(room[-1 if shift == 0 else 0]) == 7.0
    y = torch.full((T, H), 5.0, dtype=torch.bfloat16, device="cuda")
    fb.unsort_tokens(out, o, output=y)
    sums, mag = R.unsort(out, pick_row.cuda(), None)
    R.check(y, sums, K * U * mag, "y")


@pytest.mark.gpu
def test_captured_and_replayed_on_another_stream():
    """The whole run captured once, replayed with other picks, weights and tokens."""
    T, K, E, H = 700, 8, 64, 96
    g = torch.Generator().manual_seed(4)
    ids = _ids(T, K, E, 0, E, 1).cuda()
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    w = torch.rand(T, K, generator=g).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            o = fb.sort_by_expert(ids, E)
            y = fb.unsort_tokens(fb.sort_tokens(x, o), o, w)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        o = fb.sort_by_expert(ids, E)
        y = fb.unsort_tokens(fb.sort_tokens(x, o), o, w)
    for seed in (11, 12):
        ids.copy_(_ids(T, K, E, 0, E, seed))
        x.copy_(torch.randn(T, H, generator=g))
        w.copy_(torch.rand(T, K, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref = x.double() * w.double().sum(1, keepdim=True)
        mag = x.double().abs() * w.double().sum(1, keepdim=True)
        R.check(y, ref, K * U * mag, "y")


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    o = fb.sort_by_expert(ids, 4)
    x = torch.zeros((4, 8), device="cuda")
    with pytest.raises(TypeError, match="int32"):
        fb.sort_by_expert(ids.long(), 4)
    with pytest.raises(ValueError, match="contiguous"):
        fb.sort_by_expert(torch.zeros((2, 4), dtype=torch.int32, device="cuda").t(), 4)
    for kw in (dict(num_local_experts=0), dict(num_local_experts=1025),
               dict(num_local_experts=4, local_expert_offset=-1),
               dict(num_local_experts=4, align=0), dict(num_local_experts=4, align=1025)):
        with pytest.raises(ValueError):
            fb.sort_by_expert(ids, **kw)
    with pytest.raises(ValueError, match="shape"):
        fb.sort_tokens(x[:3], o)
    with pytest.raises(ValueError, match="contiguous"):
        fb.sort_tokens(torch.zeros((4, 16), device="cuda")[:, ::2], o)
    with pytest.raises(ValueError, match="shape"):
        fb.unsort_tokens(x, o)                                   # 8 rows are wanted
    rows = torch.zeros((8, 8), device="cuda")
    with pytest.raises(TypeError):
        fb.unsort_tokens(rows.to(torch.int8), o)
    with pytest.raises(ValueError, match="topk_weights"):
        fb.unsort_tokens(rows, o, torch.zeros((4, 3), device="cuda"))
    with pytest.raises(TypeError, match="topk_weights"):
        fb.unsort_tokens(rows, o, torch.zeros((4, 2), device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="gradients"):
        fb.sort_tokens(x.clone().requires_grad_(), o, output=rows)
    room = torch.zeros((12, 8), device="cuda")
    with pytest.raises(RuntimeError, match="SHAPE"):
        fb.sort_tokens(room[:4], o, output=room[2:10])           # overlapping
    with pytest.raises(TypeError, match="ExpertOrder"):
        fb.sort_tokens(x, None)


def test_refusals_on_the_host():
    with pytest.raises(ValueError, match="CUDA"):
        fb.sort_by_expert(torch.zeros((4, 2), dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="shape"):
        fb.sort_by_expert(torch.zeros(4, dtype=torch.int32), 4)
    lib = _lib.load()
    rows, scratch = ctypes.c_int64(), ctypes.c_size_t()

    def size(*a):
        return lib.fmoe_sort_size(*a, ctypes.byref(rows), ctypes.byref(scratch))
    assert size(4, 2, 4, 16) == 0 and rows.value == 8 + 4 * 15 and scratch.value == 0
    assert size(1, 2, 64, 16) == 0 and rows.value == 2 + 2 * 15
    assert size(4096, 8, 256, 1) == 0 and rows.value == 32768 and scratch.value == 0
    assert size(16384, 8, 256, 1) == 0 and rows.value == 131072 and scratch.value > 0
    assert size(4096, 8, 257, 1) == 0 and scratch.value > 0
    for bad in ((-1, 2, 4, 1), (4, 0, 4, 1), (4, 2, 0, 1), (4, 2, 1025, 1), (4, 2, 4, 0),
                (4, 2, 4, 1025), (2 ** 28, 8, 4, 1)):
        assert size(*bad) == -2, bad
    o = _lib.FmoeTokenOrder(4, 2, 4, 8, 4096, 8192, 12288)
    ref = ctypes.byref(o)
    assert lib.fmoe_sort_by_expert(None, 0, 1, None, None, 0, None) == -1
    assert lib.fmoe_sort_by_expert(None, 0, 1, ref, None, 0, None) == -1
    assert lib.fmoe_sort_by_expert(16, -1, 1, ref, None, 0, None) == -4
    assert lib.fmoe_sort_by_expert(16, 0, 16, ref, None, 0, None) == -2      # 8 rows are too few
    assert lib.fmoe_sort_by_expert(18, 0, 1, ref, None, 0, None) == -3
    assert lib.fmoe_sort_by_expert(8192, 0, 1, ref, None, 0, None) == -2     # overlaps row_pick
    big = _lib.FmoeTokenOrder(16384, 8, 4, 131072, 1 << 20, 2 << 20, 3 << 20)
    assert lib.fmoe_sort_by_expert(16, 0, 1, ctypes.byref(big), None, 0, None) == -5
    few = _lib.FmoeTokenOrder(4, 2, 4, 7, 4096, 8192, 12288)
    assert lib.fmoe_sort_rows(16, 8, ctypes.byref(few), 1 << 20, 1, None) == -2
    assert lib.fmoe_sort_rows(None, 8, ref, 1 << 20, 1, None) == -1
    assert lib.fmoe_sort_rows(16, 0, ref, 1 << 20, 1, None) == -2
    assert lib.fmoe_sort_rows(16, 8, ref, 24, 1, None) == -2                 # overlap
    assert lib.fmoe_unsort_rows(16, 7, 8, ref, None, 1 << 20, None) == -6
    assert lib.fmoe_unsort_rows(None, 0, 8, ref, None, 1 << 20, None) == -1
    assert lib.fmoe_unsort_rows(18, 0, 8, ref, None, 1 << 20, None) == -3
    assert lib.fmoe_unsort_rows_backward(16, None, 0, 8, ref, None, 1 << 20, 1 << 21, None) == -1
    assert lib.fmoe_unsort_rows_backward(16, None, 0, 8, ref, None, None, None, None) == 0
    assert ExpertOrder.__slots__
