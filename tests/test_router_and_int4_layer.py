"""Layer norm, the router's balance loss and experts of 4-bit weights as they are used: one after the
other in a layer, in graphs, from several host threads, in a training step, on tensors beyond 2^31
elements; what they refuse; and the C structs they pass."""
import ctypes
import os
import subprocess
import sys
import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from tests import layer_refs as R
from tests.conftest import ROOT
from tests.test_int4 import _expert_check, _unpack
from tests.test_layer_norm import _ref as norm_ref

HEADER = os.path.join(ROOT, "include", "fmoe.h")


def test_struct_layouts_match_c(tmp_path):
    structs = {"FmoeLayerNormArgs": _lib.FmoeLayerNormArgs, "FmoeBalanceArgs": _lib.FmoeBalanceArgs,
               "FmoeInt4Args": _lib.FmoeInt4Args}
    prog = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    want = []
    for name, s in structs.items():
        prog.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(s))
        for f, _ in s._fields_:
            prog.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(s, f).offset)
    prog.append("return 0;}")
    c, exe = tmp_path / "l.c", tmp_path / "l"
    c.write_text("\n".join(prog))
    subprocess.run(["gcc", "-std=c99", str(c), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in out.split()] == want


def _layer(x, branch, w, b, router, w1, w2, top_k):
    """An expert layer of 4-bit experts: norm, routing, two products per expert, and back."""
    hidden, normed = fb.layer_norm(branch, x, weight=w, bias=b)
    logits = normed.float() @ router.t()
    ids = logits.topk(top_k, 1).indices.to(torch.int32)
    weights = torch.softmax(logits.gather(1, ids.long()), 1)
    E = w1[0].shape[0]
    order = fb.sort_by_expert(ids, E)
    rows = fb.sort_tokens(normed, order)
    up = fb.int4_expert_matmul(rows, w1[0], w1[1], order.expert_base, w1[2], group=64)
    half = up.shape[1] // 2
    act = torch.nn.functional.silu(up[:, half:]) * up[:, :half]
    down = fb.int4_expert_matmul(act, w2[0], w2[1], order.expert_base, w2[2], group=64)
    y = fb.unsort_tokens(down, order, weights)
    out, q8 = fb.layer_norm(y, hidden, weight=w, bias=b, quantize=True)
    counts = fb.expert_counts(ids, E)
    return dict(hidden=hidden, normed=normed, order=order, rows=rows, up=up, act=act, down=down, y=y,
                weights=weights, out=out, q8=q8, counts=counts, ids=ids)


def _inputs(T, H, I, E, seed, dtype=torch.bfloat16, symmetric=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, branch = rand(T, H).to(dtype), rand(T, H).to(dtype)
    w, b = (1 + 0.1 * rand(H)).to(dtype), (0.1 * rand(H)).to(dtype)
    w1 = fb.quantize_int4((0.05 * rand(E, 2 * I, H)).to(dtype), group=64, symmetric=symmetric)
    w2 = fb.quantize_int4((0.05 * rand(E, H, I)).to(dtype), group=64, symmetric=symmetric)
    return [x, branch, w, b, rand(E, H), w1, w2]


KEYS = ("hidden", "normed", "up", "down", "y", "out", "counts")


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,I,E,top_k,dtype,symmetric", [
    (1, 256, 96, 8, 2, "bf16", True), (37, 512, 160, 16, 4, "fp16", False),
    (700, 384, 128, 4, 2, "bf16", False), (300, 256, 64, 32, 8, "fp16", True)])
def test_layer_stage_by_stage(T, H, I, E, top_k, dtype, symmetric):
    """Each operator of the chain against its definition on what the one before returned."""
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    args = _inputs(T, H, I, E, T, dt, symmetric)
    x, branch, w, b, _, w1, w2 = args
    r = _layer(*args, top_k)
    h, y, *_, = norm_ref(branch, x, w, b, 1e-5)
    R.check(r["hidden"], h, R.U * h.abs(), "hidden")
    R.check(r["normed"], y, norm_ref(branch, x, w, b, 1e-5)[4], "normed")
    order = r["order"]
    R.check(r["rows"], R.rows_of(r["normed"], order.row_pick.tolist(), top_k), 0.0, "rows")
    _expert_check(r["up"], r["rows"], *w1, 64, order.expert_base)
    _expert_check(r["down"], r["act"], *w2, 64, order.expert_base)
    ref, mag = R.unsort(r["down"], order.pick_row, r["weights"])
    R.check(r["y"], ref, (top_k + 1) * R.U * mag, "y")
    h = r["hidden"].double() + r["y"].double()
    R.check(r["out"], h, R.U * h.abs(), "out")
    assert torch.equal(r["counts"].long(), torch.bincount(r["ids"].view(-1).long(), minlength=E))
    assert fb.int4_status() == 0


@pytest.mark.gpu
def test_layer_captured_and_replayed():
    """The layer in graphs on two streams, replayed with other inputs at the same time: the bits of eager
    calls."""
    graphs = []
    for seed, T in ((1, 5), (2, 300)):
        args = _inputs(T, 512, 128, 8, seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _layer(*args, 2)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = _layer(*args, 2)
        graphs.append((graph, s, args, got, T))
    for round_ in range(3):
        for _, _, args, _, T in graphs:
            for old, new in zip(args[:5], _inputs(T, 512, 128, 8, 10 + round_)[:5]):
                old.copy_(new)
        torch.cuda.synchronize()
        for graph, s, *_ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, args, got, _ in graphs:
            want = _layer(*args, 2)
            for k in KEYS:
                assert torch.equal(got[k], want[k]), k
            assert torch.equal(got["q8"][0].view(torch.uint8), want["q8"][0].view(torch.uint8))


@pytest.mark.gpu
def test_layer_from_several_threads_at_once():
    args = [_inputs(T, 512, 128, 8, 30 + T) for T in (2, 40, 300, 64)]
    want = [_layer(*a, 2) for a in args]
    torch.cuda.synchronize()
    got = [None] * len(args)

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                r = _layer(*args[i], 2)
            s.synchronize()
        got[i] = r

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(args))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        for k in KEYS:
            assert torch.equal(g[k], w[k]), k


def _plain_step(d, ids, base, coef):
    """The training step below in the arguments' type."""
    x, branch, w, b, router, W = d
    h = x + branch
    c = h - h.mean(1, keepdim=True)
    n = c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-5) * w + b
    logits = n @ router.t()
    weights = torch.softmax(logits.gather(1, ids.long()), 1)
    per = torch.einsum("th,tkgh->tkg", n, W[ids.long()])
    y = (weights[:, :, None] * per).sum(1)
    p = torch.softmax(logits, 1)
    loss = 0.0
    E, K = router.shape[0], ids.shape[1]
    for a, e in zip(base[:-1], base[1:]):
        f = torch.bincount(ids[a:e].reshape(-1).long(), minlength=E).to(x.dtype) * E / (K * (e - a))
        loss = loss + (f * p[a:e].mean(0)).sum() / (len(base) - 1)
    return h + y, coef * loss


@pytest.mark.gpu
def test_training_step_with_the_balance_loss():
    """Norm, router, balance loss per sequence, experts (torch) and back: the gradients of every leaf
    against the same layer in 64 bits."""
    T, H, E, K = 60, 64, 8, 2
    g = torch.Generator().manual_seed(0)

    def leaf(*shape, scale=1.0, base=0.0):
        return (base + scale * torch.randn(*shape, generator=g)).cuda().requires_grad_()
    leaves = [leaf(T, H), leaf(T, H), leaf(H, scale=0.1, base=1), leaf(H, scale=0.1),
              leaf(E, H, scale=0.2), leaf(E, H, H, scale=0.1)]
    x, branch, w, b, router, W = leaves
    up, base, coef = torch.randn(T, H, generator=g).cuda(), [0, 25, 26, 60], 10.0
    seq = torch.tensor(base, dtype=torch.int32, device="cuda")

    h, normed = fb.layer_norm(branch, x, weight=w, bias=b)
    logits = normed @ router.t()
    ids = logits.detach().topk(K, 1).indices.to(torch.int32)
    loss, counts = fb.balance_loss(logits, ids, sequence_base=seq)
    weights = torch.softmax(logits.gather(1, ids.long()), 1)
    order = fb.sort_by_expert(ids, E)
    rows = fb.sort_tokens(normed, order)
    bases = order.expert_base.tolist()
    out = torch.cat([rows[i:j] @ W[e].t() for e, (i, j) in enumerate(zip(bases, bases[1:]))])
    total = h + fb.unsort_tokens(out, order, weights)
    got = torch.autograd.grad((total, coef * loss), leaves, (up, torch.ones((), device="cuda")))
    assert int(counts.sum()) == T * K

    d = [t.detach().double().requires_grad_() for t in leaves]
    y, l64 = _plain_step(d, ids, base, coef)
    ref = torch.autograd.grad((y, l64), d, (up.double(), torch.ones((), dtype=torch.float64,
                                                                     device="cuda")))
    # fp32 throughout: sums of up to T * K * H = 7680 terms and a chain of five operators stay within
    # 2^-24 * (7680^0.5 * 50) of the largest gradient of each leaf, about 2.6e-4
    for a, r in zip(got, ref):
        assert float((a.double() - r).abs().max()) <= 2.6e-4 * float(r.abs().max())


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements or bytes: the last rows are right."""
    bf = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(0)
    # 4-bit weights of 2.7e9 bytes; few rows and many rows per expert
    E, N, K = 40, 8192, 16384
    packed = torch.empty((E, N, K // 2), dtype=torch.uint8, device="cuda")
    for e in range(E):
        packed[e] = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (torch.rand(E, N, K // 128, generator=g, device="cuda") * 0.01).to(bf)
    for per in (2, 40):
        x = torch.randn(per * E, K, generator=g, device="cuda").to(bf)
        base = torch.arange(E + 1, dtype=torch.int32, device="cuda") * per
        y = fb.int4_expert_matmul(x, packed, scale, base)
        one = fb.int4_expert_matmul(x[-per:].contiguous(), packed[-1:].contiguous(),
                                    scale[-1:].contiguous(), base[:2].contiguous())
        # the same numbers, in other tiles: fp32 sums of K terms either way
        d = (y[-per:].double() - one.double()).abs()
        lim = x[-per:].double().abs().sum(1, keepdim=True) * 0.08 * (K + 40) * 2 * R.U
        assert bool((d <= lim + 2 ** -7 * one.double().abs()).all())
    back = fb.dequantize_int4(packed[20:], scale[20:].contiguous())     # 2.7e9 elements
    last = _unpack(packed[-1, -1]).float() - 8
    assert torch.equal(back[-1, -1], (last * scale[-1, -1].float().repeat_interleave(128)).to(bf))
    p2, s2, _ = fb.quantize_int4(back)
    p1, s1, _ = fb.quantize_int4(back[-1].contiguous())
    assert torch.equal(p2[-1], p1) and torch.equal(s2[-1], s1)
    del packed, scale, back, p2, s2, y, one
    # outputs of 2.4e9 elements
    M, N, K = 300000, 8192, 64
    x = torch.randn(M, K, generator=g, device="cuda").to(bf)
    p, s, _ = fb.quantize_int4((0.1 * torch.randn(N, K, generator=g, device="cuda")).to(bf), group=64)
    y = fb.int4_matmul(x, p, s, group=64)
    assert torch.equal(y[-300:], fb.int4_matmul(x[-600:].contiguous(), p, s, group=64)[-300:])
    # norms of those rows, with gradients
    y.requires_grad_()
    w = torch.ones(N, device="cuda", requires_grad=True)
    h, n = fb.layer_norm(None, y, weight=w)
    part = y.detach()[-200:].clone().requires_grad_()
    _, np_ = fb.layer_norm(None, part, weight=w)
    assert torch.equal(n.detach()[-200:], np_.detach())
    (dy,) = torch.autograd.grad(n, y, n.detach())
    (dp,) = torch.autograd.grad(np_, part, np_.detach())
    assert torch.equal(dy[-200:], dp)
    del y, h, n, dy, x
    # logits of 2.4e9 elements
    T, E = 2400000, 1024
    logits = torch.randn(T, E, generator=g, device="cuda", dtype=bf).requires_grad_()
    ids = torch.randint(0, E, (T, 2), generator=g, device="cuda", dtype=torch.int32)
    base = torch.tensor([0, T - 100, T], dtype=torch.int32, device="cuda")
    loss, counts = fb.balance_loss(logits, ids, sequence_base=base)
    (d,) = torch.autograd.grad(loss, logits)
    leaf = logits.detach()[-100:].clone().requires_grad_()
    _, c = fb.balance_loss(leaf, ids[-100:].contiguous())
    assert torch.equal(counts[1], c)
    (dl,) = torch.autograd.grad(fb.balance_loss(leaf, ids[-100:].contiguous())[0], leaf,
                                torch.tensor(0.5, device="cuda"))       # the mean of two sequences
    assert torch.equal(d[-100:], dl)


@pytest.mark.gpu
def test_dual_tensors_are_refused():
    x, y, w = (torch.randn(*s, device="cuda") for s in ((4, 64), (4, 64), (64,)))
    ids = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    xh = x.half()
    p, s, _ = fb.quantize_int4(xh, group=64)
    calls = [(lambda t: fb.layer_norm(t, y, weight=w), x), (lambda t: fb.layer_norm(None, t), x),
             (lambda t: fb.layer_norm(x, y, weight=t), w), (lambda t: fb.layer_norm(x, y, bias=t), w),
             (lambda t: fb.balance_loss(t, ids)[0], x), (lambda t: fb.quantize_int4(t, group=64)[1], x),
             (lambda t: fb.dequantize_int4(p, t, group=64), s),
             (lambda t: fb.int4_matmul(t, p, s, group=64), xh),
             (lambda t: fb.int4_matmul(xh, p, t, group=64), s),
             (lambda t: fb.int4_matmul(xh, p, s, None, t, group=64), w[:4].contiguous())]
    for call, t in calls:
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            call(t)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("call", [
    lambda x: fb.layer_norm(None, x), lambda x: fb.balance_loss(x, x)[0],
    lambda x: fb.expert_counts(x, 4), lambda x: fb.quantize_int4(x)[0],
    lambda x: fb.dequantize_int4(x, x), lambda x: fb.int4_matmul(x, x, x),
    lambda x: fb.int4_expert_matmul(x, x, x, x)])
def test_tracing_is_refused(call):
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, torch.ones(4, 8))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(torch.ones(4, 8))


@pytest.mark.gpu
def test_a_changed_input_is_noticed_by_the_backward_pass():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    logits = (x * 2)
    loss, counts = fb.balance_loss(logits, torch.zeros((4, 1), dtype=torch.int32, device="cuda"))
    counts.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    f = x * 3
    _, n = fb.layer_norm(f, x)
    with torch.no_grad():
        f.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        n.sum().backward()


def test_counts_that_pass_int32_are_refused():
    """2^31 picks and more: the counts are int32. Shapes alone, nothing is read."""
    lib, P = _lib.load(), 1 << 20
    for T, K, rc in ((2 ** 30, 2, -2), (2 ** 30 + 1, 4, -2), (5, 2 ** 31 - 1, -2), (2 ** 30 - 1, 2, -5)):
        a = _lib.FmoeBalanceArgs(T, 4, K, 1, _lib.DTYPE_BF16, 0, P, P, None, P, P, P)
        assert lib.fmoe_balance_loss(ctypes.byref(a), None) == rc        # -5: no workspace


def test_groups_that_pass_int32_are_refused():
    lib, P = _lib.load(), 1 << 20
    for group in (2 ** 31 - 128, 2 ** 31 - 131072, 0, -128, 48, 96):
        assert lib.fmoe_quantize_int4(P, 1, 4, 256, group, 2 * P, 3 * P, None, None) == -2
        assert lib.fmoe_dequantize_int4(P, 2 * P, 1, None, 4, 256, group, 3 * P, 1, None) == -2
        a = _lib.FmoeInt4Args(1, 8, 256, 1, group, 1, 1, P, 2 * P, 3 * P, None, None, None, 4 * P, 0)
        assert lib.fmoe_int4_matmul(ctypes.byref(a), None) == -2


def test_the_packed_solution_imports_on_its_own(tmp_path):
    """The modules that the package imports are all among those that the solution packs."""
    from flashinfer_b200 import solution
    dest = tmp_path / "sol"
    solution.unpack(solution.pack(), str(dest))
    code = ("import flashinfer_b200 as f; print(f.__file__, f.balance_loss.__module__, "
            "f.int4_matmul.__module__, f.layer_norm.__module__)")
    r = subprocess.run([sys.executable, "-c", code], cwd=dest, capture_output=True, text=True,
                       env={**os.environ, "PYTHONPATH": str(dest)})
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.startswith(str(dest))
