"""Calls at the edges of what the operators around the experts allow: empty batches in tables of a fixed
size, autograd modes, given outputs, hand-made orders, sizes beyond 32 bits."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import flashinfer_b200 as fb
from flashinfer_b200 import _lib, _op


def _order_struct(T, K, E, R, base=4096, row_pick=8192, pick_row=12288):
    return ctypes.byref(_lib.FmoeTokenOrder(T, K, E, R, base, row_pick, pick_row))


def test_rows_without_tokens_need_their_table():
    """No tokens but rows: the kernels write and read row_pick, so it must be there."""
    lib = _lib.load()
    o = _order_struct(0, 2, 4, 8, row_pick=None, pick_row=None)
    assert lib.fmoe_sort_by_expert(None, 0, 1, o, None, 0, None) == -1
    assert lib.fmoe_sort_rows(None, 8, o, 1 << 20, 1, None) == -1
    assert lib.fmoe_unsort_rows(1 << 20, 0, 8, o, None, None, None) == -1
    assert lib.fmoe_unsort_rows_backward(None, None, 0, 8, o, None, 1 << 20, None, None) == -1
    # neither tokens nor rows: nothing to read
    none = _order_struct(0, 2, 4, 0, row_pick=None, pick_row=None)
    assert lib.fmoe_sort_rows(None, 8, none, None, 1, None) == 0
    assert lib.fmoe_unsort_rows(None, 0, 8, none, None, None, None) == 0


@pytest.mark.gpu
def test_no_tokens_in_tables_of_a_fixed_size():
    """Zero tokens and eight rows: the order says that no row holds a pick, sorted rows are zero with
    zero_tail and left alone without."""
    lib = _lib.load()
    stream = torch.cuda.current_stream().cuda_stream
    base = torch.full((5,), 7, dtype=torch.int32, device="cuda")
    row_pick = torch.full((8,), 7, dtype=torch.int32, device="cuda")
    o = _order_struct(0, 2, 4, 8, base.data_ptr(), row_pick.data_ptr(), None)
    assert lib.fmoe_sort_by_expert(None, 0, 1, o, None, 0, stream) == 0
    assert base.tolist() == [0] * 5 and row_pick.tolist() == [-1] * 8
    rows = torch.full((8, 6), 3.0, device="cuda")
    assert lib.fmoe_sort_rows(None, 24, o, rows.data_ptr(), 0, stream) == 0
    assert bool((rows == 3.0).all())
    assert lib.fmoe_sort_rows(None, 24, o, rows.data_ptr(), 1, stream) == 0
    assert not bool(rows.any())


@pytest.mark.gpu
@pytest.mark.parametrize("tag,dtype", [(0, torch.float32), (1, torch.bfloat16)])
def test_gradient_of_rows_without_tokens_is_zero(tag, dtype):
    """Every row's gradient is written, also where a batch of no tokens meets a table of a fixed size."""
    lib = _lib.load()
    stream = torch.cuda.current_stream().cuda_stream
    base = torch.zeros(5, dtype=torch.int32, device="cuda")
    row_pick = torch.full((8,), -1, dtype=torch.int32, device="cuda")
    o = _order_struct(0, 2, 4, 8, base.data_ptr(), row_pick.data_ptr(), None)
    flat = torch.full((8 * 33 + 2,), 3.0, dtype=dtype, device="cuda")
    grad = flat[1:-1]
    assert lib.fmoe_unsort_rows_backward(None, None, tag, 33, o, None, grad.data_ptr(), None,
                                         stream) == 0
    assert not bool(grad.any()) and float(flat[0]) == 3.0 and float(flat[-1]) == 3.0
    assert lib.fmoe_unsort_rows_backward(None, None, tag, 33, o, None, grad.data_ptr() + 1, None,
                                         stream) == -3


def _int8_calls():
    """The int8 operators' calls and, for each, the float tensors that it takes."""
    x = torch.randn(4, 32, device="cuda").to(torch.bfloat16)
    a = torch.ones((4, 32), dtype=torch.int8, device="cuda")
    w = torch.ones((6, 32), dtype=torch.int8, device="cuda")
    s4, s6, bias = (torch.ones(n, device="cuda") for n in (4, 6, 6))
    out = torch.zeros((4, 6), device="cuda")
    base = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    return [(lambda: fb.quantize_int8(x), (x,)),
            (lambda: fb.int8_matmul(a, w, s4, s6, bias, output=out), (s4, s6, bias, out)),
            (lambda: fb.int8_expert_matmul(a, w[None], s4, s6[None], base, output=out),
             (s4, s6, out))]


@pytest.mark.gpu
def test_int8_operators_are_not_recorded():
    """A float tensor that requires a gradient is refused, unless nothing is recorded."""
    for call, tensors in _int8_calls():
        call()
        for t in tensors:
            t.requires_grad_()
            with pytest.raises(ValueError, match="no gradient"):
                call()
            with torch.no_grad():
                call()
            with torch.inference_mode():
                call()
            t.requires_grad_(False)
        call()


def test_dual_tensors_are_refused():
    """A dual tensor does not require a gradient, but a result without a tangent would be wrong."""
    t = torch.ones(3)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(t, t)
        assert not _op.recording(t, None)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                _op.recording(t, None, d)
    assert not _op.recording(t, None)


@pytest.mark.gpu
def test_dual_tensors_are_refused_by_every_operator():
    order = fb.sort_by_expert(torch.zeros((4, 1), dtype=torch.int32, device="cuda"), 1)
    x, y, w = (torch.randn(*s, device="cuda") for s in ((4, 32), (4, 32), (32,)))
    weights = torch.rand(4, 1, device="cuda")
    calls = [(lambda x: fb.block_norm(x, y, post_weight=w, pre_weight=w), x),
             (lambda x: fb.block_norm(y, x, pre_weight=w), x),
             (lambda p: fb.block_norm(x, y, post_weight=p), w),
             (lambda p: fb.block_norm(x, y, gate=p), w),
             (lambda p: fb.block_norm(x, y, pre_weight=p), w),
             (lambda x: fb.sort_tokens(x, order), x),
             (lambda x: fb.unsort_tokens(x, order, weights), x),
             (lambda p: fb.unsort_tokens(x, order, p), weights),
             (lambda x: fb.quantize_int8(x.to(torch.bfloat16)), x)]
    for call, t in calls:
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            call(t)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("call", [
    lambda x: fb.block_norm(None, x, pre_weight=x[0]), lambda x: fb.quantize_int8(x),
    lambda x: fb.sort_by_expert(x, 4).expert_base, lambda x: fb.sort_tokens(x, None),
    lambda x: fb.unsort_tokens(x, None), lambda x: fb.int8_matmul(x, x, x, x),
    lambda x: fb.int8_expert_matmul(x, x, x, x, x)])
def test_tracing_is_refused(call):
    """Before anything else is looked at: a trace would return memory that nothing wrote."""
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, torch.ones(4, 8))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(torch.ones(4, 8))


@pytest.mark.gpu
def test_other_dispatch_modes_are_left_alone():
    class Pass(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x = torch.randn(4, 32, device="cuda")
    want = fb.block_norm(None, x, pre_weight=x[0])[1]
    with Pass():
        assert torch.equal(fb.block_norm(None, x, pre_weight=x[0])[1], want)


def test_an_order_of_host_tables_is_refused():
    base, rows = torch.zeros(5, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fb.ExpertOrder(base, rows, torch.zeros((4, 2), dtype=torch.int32))
    with pytest.raises(ValueError, match="axes"):
        fb.ExpertOrder(base, rows, rows)
    with pytest.raises(TypeError, match="Tensor"):
        fb.ExpertOrder(base, rows, None)


@pytest.mark.gpu
def test_the_tables_of_an_order_are_checked_and_stay():
    """A hand-made order is checked as every argument is; its attributes cannot be set, since the library
    would keep the old table's address."""
    ids = torch.tensor([[0, 3], [1, 0], [2, 2], [3, 1]], dtype=torch.int32, device="cuda")
    made = fb.sort_by_expert(ids, 4)
    base, rows, picks = made.expert_base, made.row_pick, made.pick_row
    order = fb.ExpertOrder(base, rows, picks)
    x = torch.randn(4, 8, device="cuda")
    assert torch.equal(fb.sort_tokens(x, order), fb.sort_tokens(x, made))
    assert (order.num_tokens, order.top_k, order.num_rows) == (4, 2, 8)
    assert order.device == x.device
    for name in ("expert_base", "row_pick", "pick_row", "num_tokens", "top_k", "num_rows", "device"):
        with pytest.raises(AttributeError):
            setattr(order, name, getattr(order, name))
    for bad in ((base.long(), rows, picks), (base, rows.long(), picks), (base, rows, picks.long())):
        with pytest.raises(TypeError, match="int32"):
            fb.ExpertOrder(*bad)
    for bad in ((base.cpu(), rows, picks), (base, rows.cpu(), picks),
                (base, rows.repeat(2)[::2], picks), (base, rows, picks.t()), (base, rows[:7], picks),
                (base[:1], rows, picks), (base[None], rows, picks), (base, rows[None], picks)):
        with pytest.raises(ValueError):
            fb.ExpertOrder(*bad)


@pytest.mark.gpu
def test_a_given_output_counts_as_changed():
    """A tensor that a recorded operation saved and a later call writes to: the backward pass raises, as
    it does for torch's own operations in place."""
    order = fb.sort_by_expert(torch.zeros((4, 1), dtype=torch.int32, device="cuda"), 1)
    x, y, w = (torch.randn(*s, device="cuda") for s in ((4, 32), (4, 32), (32,)))
    a = torch.ones((4, 32), dtype=torch.int8, device="cuda")
    b = torch.ones((32, 32), dtype=torch.int8, device="cuda")
    s4, s32 = torch.ones(4, device="cuda"), torch.ones(32, device="cuda")
    base = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    calls = [lambda o: fb.block_norm(x, o, pre_weight=w, output=o)[0],       # in place
             lambda o: fb.block_norm(x, y, output=o)[0],
             lambda o: fb.sort_tokens(x, order, output=o),
             lambda o: fb.unsort_tokens(x, order, output=o),
             lambda o: fb.int8_matmul(a, b, s4, s32, output=o),
             lambda o: fb.int8_expert_matmul(a, b[None], s4, s32[None], base, output=o)]
    for call in calls:
        out = torch.randn(4, 32, device="cuda")
        p = torch.ones(4, 32, device="cuda", requires_grad=True)
        loss = (p * out).sum()
        before = out._version
        with torch.no_grad():
            assert call(out) is out
        assert out._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            call(torch.zeros(4, 32, device="cuda"))


@pytest.mark.gpu
def test_an_offset_beyond_32_bits_is_refused():
    """As a C int it would be another offset: 2^32 would name expert 0."""
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    last = fb.sort_by_expert(ids, 4, 2 ** 31 - 1)
    assert last.expert_base.tolist() == [0] * 5 and bool((last.pick_row == -1).all())
    for offset in (2 ** 31, 2 ** 32, 2 ** 32 + 3, -1):
        with pytest.raises(ValueError, match="local_expert_offset"):
            fb.sort_by_expert(ids, 4, offset)


def test_channels_beyond_32_bits_are_refused():
    from flashinfer_b200.int8 import _check_sizes
    _check_sizes(2 ** 31 - 1, 16)
    for channels in (2 ** 31, 2 ** 32 + 8):
        with pytest.raises(ValueError, match="channels"):
            _check_sizes(channels, 16)


@pytest.mark.gpu
def test_picks_beyond_32_bits_are_refused():
    """2^32 + 4 tokens: as a C int four. The tensor is only allocated (17 GB), and read by nothing."""
    ids = torch.empty((2 ** 32 + 4, 1), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="picks"):
        fb.sort_by_expert(ids, 4)


@pytest.mark.gpu
def test_rows_of_conjugate_views():
    """Rows of any type, complex ones among them: a conjugate view shares the bytes of its base."""
    ids = torch.tensor([[0, 3], [1, 0], [2, 2], [3, 1]], dtype=torch.int32, device="cuda")
    order = fb.sort_by_expert(ids, 4)
    x = torch.randn(4, 5, dtype=torch.complex64, device="cuda")
    want = fb.sort_tokens(x.conj().resolve_conj(), order)
    assert torch.equal(want[:, 0], x.conj()[order.row_pick.long() // 2][:, 0])
    assert torch.equal(fb.sort_tokens(x.conj(), order), want)
    out = torch.empty_like(want)
    assert torch.equal(fb.sort_tokens(x.conj(), order, output=out), want)
    with pytest.raises(ValueError, match="conjugate"):
        fb.sort_tokens(x, order, output=out.conj())
