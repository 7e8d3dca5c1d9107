"""The router's balance loss, its counts and its gradient, against the definition in 64 bits."""
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


def _inputs(T, E, K, dtype, seed=0, spread=1.0):
    g = _gen(seed + 7 * T + E)
    logits = (spread * (torch.randn(T, E, generator=g, device="cuda")
                        + 0.7 * torch.randn(E, generator=g, device="cuda"))).to(dtype)
    ids = torch.randint(-1, E + 1, (T, K), generator=g, device="cuda", dtype=torch.int32)
    return logits, ids


def _spans(base, T):
    """Rows of every sequence: bases clamped to [0, T] and taken as a running maximum."""
    most, clean = 0, []
    for b in base:
        most = max(most, min(max(b, 0), T))
        clean.append(most)
    return list(zip(clean[:-1], clean[1:]))


def _ref(logits, ids, scoring, base=None):
    """loss, counts, gradient, and the bounds of loss and gradient.

    A score's exponential has a relative error of 4 U (expf: two units) and what the rounding of its
    argument adds, U |l - max|; a sigmoid at most 10 U (1 + exp, a division of two units, a product). Its
    row sum adds 37 U (32 values in a lane, 5 levels) and the weighted errors of the terms, the
    reciprocal and the product 2 U each. A sum over rows has at most T + 80 additions (a warp's rows, eight
    warps, the blocks in 32 parts). In the gradient c is within 4 U, the dot product adds 37 U.
    """
    z = logits.double()
    T, E = z.shape
    K = ids.shape[1]
    top = z.amax(1, keepdim=True)
    live = torch.isfinite(top)
    if scoring == "softmax":
        e = torch.where(live, torch.exp(z - torch.where(live, top, 0.0)), 0.0)
        e_rel = 4 * U + U * torch.where(torch.isfinite(z), (z - top).abs(), 0.0)
        slope = torch.ones_like(z)
    else:
        # sigmoid(l) exp(-m), with m the row's largest logit where all are below -60
        low = (top < -60) & live
        m = torch.where(low, top, 0.0)
        e = torch.where(live, torch.sigmoid(z) if not bool(low.any())
                        else torch.where(low, torch.exp(z - m), torch.sigmoid(z)), 0.0)
        e_rel = 10 * U + torch.where(low & torch.isfinite(z), U * (z - m).abs(), 0.0)
        e_rel = e_rel + torch.where(low, torch.exp(top), 0.0)
        slope = torch.sigmoid(-z)
    total = e.sum(1, keepdim=True)
    p = torch.where(total > 0, e / total.clamp(min=1e-300), 0.0)
    p_rel = e_rel + 41 * U + (p * e_rel).sum(1, keepdim=True)
    spans = [(0, T)] if base is None else _spans(base, T)
    full = [s for s in spans if s[1] > s[0]]
    counts = torch.zeros(len(spans), E, dtype=torch.int64, device=z.device)
    loss, err = z.new_zeros(()), z.new_zeros(())
    grad, g_err = torch.zeros_like(z), torch.zeros_like(z)
    for s, (a, b) in enumerate(spans):
        if b <= a:
            continue
        picks = ids[a:b].reshape(-1).long()
        picks = picks[(picks >= 0) & (picks < E)]
        counts[s] = torch.bincount(picks, minlength=E)
        c = counts[s].double() * E / (K * (b - a) ** 2 * len(full))
        ps, rel = p[a:b], p_rel[a:b]
        loss = loss + (c * ps.sum(0)).sum()
        err = err + (c * (ps * (rel + (T + 80) * U)).sum(0)).sum()
        dot = (ps * c).sum(1, keepdim=True)
        e_dot = (ps * c * (rel + 41 * U)).sum(1, keepdim=True)
        grad[a:b] = ps * (c - dot) * slope[a:b]
        g_err[a:b] = slope[a:b] * ps * ((c - dot).abs() * (rel + 14 * U) + 5 * U * c + e_dot
                                        + 2 * U * (c + dot))
    return loss, counts, grad, err, g_err


def _check(logits, ids, scoring, base=None):
    T = logits.shape[0]
    b = None if base is None else torch.tensor(base, dtype=torch.int32, device="cuda")
    loss_ref, counts_ref, grad_ref, err, g_err = _ref(logits, ids, scoring, base)
    if base is None:
        counts_ref = counts_ref[0]
    loss, counts = fb.balance_loss(logits, ids, scoring=scoring, sequence_base=b)
    assert loss.shape == () and loss.dtype == torch.float32 and counts.dtype == torch.int32
    R.check(loss, loss_ref, err, "loss")
    assert torch.equal(counts.long(), counts_ref)
    assert torch.equal(fb.expert_counts(ids, logits.shape[1], sequence_base=b), counts)
    leaf = logits.clone().requires_grad_()
    loss2, counts2 = fb.balance_loss(leaf, ids, scoring=scoring, sequence_base=b)
    assert torch.equal(loss2.detach(), loss) and torch.equal(counts2, counts)
    g = torch.tensor(0.75 * max(T, 1), device="cuda")  # fp16 gradients of ordinary size
    (d,) = torch.autograd.grad(loss2, leaf, g)
    R.check(d, grad_ref * g.double(), g_err * g.double(), "d logits")


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K,dtype", [
    (1, 1, 1, "fp32"), (1, 256, 8, "fp32"), (2, 3, 2, "bf16"), (64, 256, 8, "fp32"),
    (33, 100, 6, "bf16"), (257, 160, 6, "fp16"), (1000, 64, 1, "bf16"), (500, 257, 4, "fp32"),
    (77, 1024, 8, "bf16"), (40, 1023, 3, "fp16"), (3001, 256, 8, "fp32"), (6000, 8, 2, "fp32")])
def test_one_sequence(T, E, K, dtype, scoring):
    _check(*_inputs(T, E, K, DT[dtype]), scoring)


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K,dtype,base", [
    (10, 16, 2, "fp32", [0, 4, 4, 9]),                  # an empty one, a row of padding
    (50, 256, 8, "bf16", [5, 6, 7, 50]),                # rows before the first, sequences of one token
    (700, 60, 4, "fp32", [0, 1, 300, 301, 301, 699]),
    (3000, 256, 8, "fp16", [0, 1000, 1008, 2990]),
    (40, 7, 2, "fp32", [0, 0, 0]),                      # none has tokens
    (40, 32, 2, "fp32", [-5, 20, 10, 30, 90]),          # steps back, and beyond both ends
    (300, 33, 3, "bf16", list(range(0, 301)))])         # one token each
def test_sequences(T, E, K, dtype, base, scoring):
    _check(*_inputs(T, E, K, DT[dtype]), scoring, base)


@pytest.mark.gpu
def test_the_most_sequences():
    T = 5000
    logits, ids = _inputs(T, 8, 2, torch.float32)
    _check(logits, ids, "softmax", [i for i in range(4096)] + [T])
    with pytest.raises(ValueError, match="4096"):
        fb.balance_loss(logits, ids, sequence_base=torch.zeros(4098, dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_masked_experts_and_far_logits(scoring, dtype):
    t = DT[dtype]
    logits, ids = _inputs(30, 48, 4, t)
    logits[3] = float("-inf")                 # nothing left
    logits[4, :40] = float("-inf")
    logits[5, 1:] = torch.finfo(t).min        # the lowest value as a mask
    logits[6] = torch.finfo(t).min
    logits[7] -= 300                          # every sigmoid out of range
    logits[8] += 300
    logits[9] = -80
    _check(logits, ids, scoring, [0, 12, 30])
    leaf = logits.clone().requires_grad_()
    loss, _ = fb.balance_loss(leaf, ids, scoring=scoring)
    (d,) = torch.autograd.grad(loss, leaf)
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(d).all())
    assert not bool(d[3].any()) and not bool(d[4, :40].any())


@pytest.mark.gpu
def test_even_use_has_loss_one():
    E = 32
    ids = torch.arange(E, dtype=torch.int32, device="cuda").view(E, 1)
    for scoring in ("softmax", "sigmoid"):
        loss, counts = fb.balance_loss(torch.zeros(E, E, device="cuda"), ids, scoring=scoring)
        assert abs(float(loss) - 1) <= 64 * U and bool((counts == 1).all())


@pytest.mark.gpu
def test_nan_is_not_hidden_and_stays_in_its_sequence():
    logits, ids = _inputs(20, 16, 2, torch.float32)
    logits[3, 5] = float("nan")
    base = torch.tensor([0, 10, 20], dtype=torch.int32, device="cuda")
    leaf = logits.requires_grad_()
    loss, _ = fb.balance_loss(leaf, ids, sequence_base=base)
    assert bool(torch.isnan(loss))
    (d,) = torch.autograd.grad(loss, leaf)
    assert bool(torch.isnan(d[3]).all())
    keep = [i for i in range(20) if i != 3]
    assert bool(torch.isfinite(d[keep]).all())


@pytest.mark.gpu
def test_no_tokens_and_no_picks():
    logits = torch.zeros((0, 16), device="cuda", requires_grad=True)
    loss, counts = fb.balance_loss(logits, torch.zeros((0, 2), dtype=torch.int32, device="cuda"))
    assert float(loss) == 0 and not bool(counts.any())
    assert torch.autograd.grad(loss, logits)[0].shape == (0, 16)
    none = torch.full((9, 2), -1, dtype=torch.int32, device="cuda")
    leaf = torch.randn(9, 16, generator=_gen(0), device="cuda").requires_grad_()
    loss, counts = fb.balance_loss(leaf, none)
    assert float(loss) == 0 and not bool(counts.any())
    assert not bool(torch.autograd.grad(loss, leaf)[0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1, 2])
def test_off_the_16_byte_boundary(off):
    logits, ids = _inputs(37, 64, 4, torch.bfloat16)
    buf = torch.zeros(37 * 64 + off, dtype=torch.bfloat16, device="cuda")
    moved = buf[off:].view(37, 64)
    moved.copy_(logits)
    _check(moved, ids, "softmax")


@pytest.mark.gpu
def test_gradient_against_differences():
    logits, ids = _inputs(12, 20, 3, torch.float32)
    base = [0, 5, 12]
    b = torch.tensor(base, dtype=torch.int32, device="cuda")
    for scoring in ("softmax", "sigmoid"):
        leaf = logits.clone().requires_grad_()
        loss, _ = fb.balance_loss(leaf, ids, scoring=scoring, sequence_base=b)
        (d,) = torch.autograd.grad(loss, leaf)
        way = torch.randn(12, 20, generator=_gen(4), device="cuda").double()
        z, step = logits.double(), 1e-6
        hi = _ref(z + step * way, ids, scoring, base)[0]
        lo = _ref(z - step * way, ids, scoring, base)[0]
        got, terms = (d.double() * way).sum(), (d.double() * way).abs().sum()
        # fp32 gradient: 1e-5 of the terms; the quotient's own error is of order 1e-10
        assert abs(float(got - (hi - lo) / (2 * step))) <= 1e-5 * float(terms) + 1e-9


@pytest.mark.gpu
def test_same_bits_again_on_streams_and_in_a_graph():
    logits, ids = _inputs(2999, 256, 8, torch.float32)
    leaf = logits.requires_grad_()
    base = torch.tensor([0, 1000, 1001, 2900], dtype=torch.int32, device="cuda")

    def step():
        loss, counts = fb.balance_loss(leaf, ids, scoring="sigmoid", sequence_base=base)
        return [loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    with torch.no_grad():
        leaf.mul_(1.5)
    ids.copy_(ids.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, step()))


@pytest.mark.gpu
def test_counts_step_a_routing_bias():
    """The counts alone: picks of a sharded range, shifted ids, more picks than rows."""
    ids = torch.randint(0, 64, (1000, 6), generator=_gen(2), device="cuda", dtype=torch.int32)
    ref = torch.bincount(ids.reshape(-1).long(), minlength=64)
    assert torch.equal(fb.expert_counts(ids, 64).long(), ref)
    assert torch.equal(fb.expert_counts(ids - 16, 20).long(), ref[16:36])
    assert torch.equal(fb.expert_counts(ids.view(1, -1), 64).long(), ref)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    logits, ids = _inputs(4, 16, 2, torch.float32)
    with pytest.raises(TypeError, match="topk_ids"):
        fb.balance_loss(logits, ids.long())
    with pytest.raises(ValueError, match="top_k"):
        fb.balance_loss(logits, ids[:3])
    with pytest.raises(ValueError, match="scoring"):
        fb.balance_loss(logits, ids, scoring="relu")
    with pytest.raises(TypeError, match="sequence_base"):
        fb.balance_loss(logits, ids, sequence_base=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="sequence_base"):
        fb.balance_loss(logits, ids, sequence_base=ids[0, :1].contiguous())
    with pytest.raises(ValueError, match="1..1024"):
        fb.balance_loss(torch.zeros((4, 1025), device="cuda"), ids)
    with pytest.raises(ValueError, match="contiguous"):
        fb.balance_loss(logits.t().contiguous().t(), ids)
    with pytest.raises(ValueError, match="num_experts"):
        fb.expert_counts(ids, 0)
    leaf = logits.clone().requires_grad_()
    loss, counts = fb.balance_loss(leaf, ids)
    assert not counts.requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, leaf, create_graph=True)


def test_refusals_on_the_host():
    with pytest.raises(ValueError, match="CUDA"):
        fb.balance_loss(torch.zeros((2, 8)), torch.zeros((2, 1), dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        fb.expert_counts(torch.zeros((2, 1), dtype=torch.int32), 8)
    lib = _lib.load()
    size = ctypes.c_size_t()
    assert lib.fmoe_balance_workspace_size(17, 8, 3, ctypes.byref(size)) == 0
    assert size.value == (3 + 3) * 8 * 8
    assert lib.fmoe_balance_workspace_size(17, 1025, 3, ctypes.byref(size)) == -2
    assert lib.fmoe_balance_workspace_size(17, 8, 4097, ctypes.byref(size)) == -2
    assert lib.fmoe_balance_workspace_size(17, 8, 3, None) == -1
    assert lib.fmoe_balance_loss(None, None) == -1
    a = _lib.FmoeBalanceArgs()

    def run(fn=lib.fmoe_balance_loss, **kw):
        a.num_tokens, a.num_experts, a.top_k, a.num_sequences = 4, 8, 2, 1
        a.dtype, a.scoring = 0, 0
        a.logits, a.topk_ids, a.sequence_base = 1 << 20, 2 << 20, None
        a.loss, a.counts, a.factor = 3 << 20, 4 << 20, 5 << 20
        a.grad_loss, a.grad_logits = 6 << 20, 7 << 20
        a.workspace, a.workspace_bytes = 8 << 20, 1 << 20
        for k, v in kw.items():
            setattr(a, k, v)
        return fn(ctypes.byref(a), None)
    for bad in ({"num_tokens": -1}, {"num_experts": 0}, {"num_experts": 1025}, {"top_k": 0},
                {"num_sequences": 0}, {"num_sequences": 2}, {"scoring": 2},
                {"sequence_base": 9 << 20, "num_sequences": 4097}):
        assert run(**bad) == -2, bad
        assert run(lib.fmoe_balance_loss_backward, **bad) == -2, bad
    assert run(dtype=3) == -6
    assert run(logits=(1 << 20) + 2) == -3 and run(counts=(4 << 20) + 1) == -3
    assert run(topk_ids=None) == -1 and run(counts=None) == -1 and run(factor=None) == -1
    assert run(workspace=None) == -5 and run(workspace_bytes=(1 + 1) * 8 * 8 - 1) == -5
    assert run(counts=2 << 20) == -2                       # counts over the picks
    back = lib.fmoe_balance_loss_backward
    assert run(back, num_tokens=0) == 0
    assert run(back, grad_loss=None) == -1 and run(back, logits=None) == -1
    assert run(back, grad_logits=1 << 20) == -2            # over the logits
