"""The operators around the experts as they are used: one after the other in a layer, in a training
step, in a captured graph, on tensors beyond 2^31 elements; and the C structs they pass."""
import ctypes
import os
import subprocess
import threading

import numpy as np
import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from flashinfer_b200 import workload as wl
from tests import layer_refs as R
from tests.conftest import ROOT
from tests.layer_refs import U

HEADER = os.path.join(ROOT, "include", "fmoe.h")


def test_struct_layouts_match_c(tmp_path):
    structs = {"FmoeTokenOrder": _lib.FmoeTokenOrder, "FmoeBlockNormArgs": _lib.FmoeBlockNormArgs}
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


def _weights(g, E, N, K):
    w = (torch.randn(E, N, K, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    q, s = fb.quantize_int8(w.view(E * N, K))
    return q.view(E, N, K), s.view(E, N)


def _layer(x, branch, post_w, gate, pre_w, logits, bias, w1, s1, w2, s2, offset):
    """One int8 expert layer: norms, routing, two products per expert, and back."""
    E = w1.shape[0]
    hidden, normed = fb.block_norm(branch, x, post_weight=post_w, gate=gate, pre_weight=pre_w)
    ids, weights = fb.route(logits, bias, 2.5)
    order = fb.sort_by_expert(ids, E, offset)
    q, scale = fb.quantize_int8(normed)
    rows, row_scale = fb.sort_tokens(q, order), fb.sort_tokens(scale, order)
    up = fb.int8_expert_matmul(rows, w1, row_scale, s1, order.expert_base)
    half = up.shape[1] // 2
    act = torch.nn.functional.silu(up[:, half:]) * up[:, :half]
    aq, a_scale = fb.quantize_int8(act)
    down = fb.int8_expert_matmul(aq, w2, a_scale, s2, order.expert_base)
    y = fb.unsort_tokens(down, order, weights)
    out, q8 = fb.block_norm(y, hidden, post_weight=post_w, pre_weight=pre_w, quantize=True)
    return dict(hidden=hidden, normed=normed, ids=ids, weights=weights, order=order, q=q,
                scale=scale, rows=rows, row_scale=row_scale, up=up, act=act, aq=aq,
                a_scale=a_scale, down=down, y=y, out=out, q8=q8)


def _layer_inputs(T, H, I, E, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    bf = torch.bfloat16
    x, branch = (torch.randn(T, H, generator=g, device="cuda").to(bf) for _ in range(2))
    post_w, pre_w = ((1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(bf)
                     for _ in range(2))
    gate = torch.rand(T, 1, generator=g, device="cuda").to(bf)
    logits = torch.randn(T, 256, generator=g, device="cuda")
    bias = (0.1 * torch.randn(256, generator=g, device="cuda")).to(bf)
    return [x, branch, post_w, gate, pre_w, logits, bias, *_weights(g, E, 2 * I, H),
            *_weights(g, E, H, I)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,I,E,offset", [(1, 256, 128, 256, 0), (37, 512, 256, 64, 96),
                                            (300, 1024, 384, 32, 224)])
def test_layer_stage_by_stage(T, H, I, E, offset):
    """Every stage of the chain against the 64-bit form of what the stage before it handed over."""
    args = _layer_inputs(T, H, I, E, T)
    x, branch, post_w, gate, pre_w, _, _, w1, s1, w2, s2 = args
    r = _layer(*args, offset)
    v = [t.double() for t in (branch, x, post_w, gate, pre_w)]
    eh, ey, *_ = R.block_norm_bounds(*v, 1.0, 1e-6)
    rh, ry = R.block_norm(*v, 1.0, 1e-6)
    R.check(r["hidden"], rh, eh, "hidden")
    R.check(r["normed"], ry, ey, "normed")
    base, row_pick, pick_row = R.order(r["ids"].cpu(), offset, E, 1)
    order = r["order"]
    assert order.expert_base.tolist() == base and torch.equal(order.pick_row.cpu(), pick_row)
    rq, rs = R.quantize(r["normed"])
    assert torch.equal(r["q"].double(), rq)
    assert torch.equal(r["rows"].double(), R.rows_of(r["q"], row_pick, 8))
    assert torch.equal(r["row_scale"].double(), R.rows_of(r["scale"][:, None], row_pick, 8)[:, 0])
    for got, a, a_s, w, s in ((r["up"], r["rows"], r["row_scale"], w1, s1),
                              (r["down"], r["aq"], r["a_scale"], w2, s2)):
        for e in range(E):
            lo, hi = base[e], base[e + 1]
            ref, err = R.product(a[lo:hi], w[e], a_s[lo:hi], s[e])
            R.check(got[lo:hi], ref, err, f"expert {e}")
        assert not bool(got[base[-1]:].any())
    ref, mag = R.unsort(r["down"], pick_row.cuda(), r["weights"])
    R.check(r["y"], ref, 8 * U * mag, "y")
    v = [r["y"].double(), r["hidden"].double(), post_w.double(), None, pre_w.double()]
    eh, ey, *_ = R.block_norm_bounds(*v, 1.0, 1e-6)
    rh, ry = R.block_norm(*v, 1.0, 1e-6)
    R.check(r["out"], rh, eh, "out")
    q8, s8 = r["q8"]
    step = s8.t().double().repeat_interleave(128, 1)
    assert bool(((q8.double() * step - ry).abs()
                 <= ey * 1.1 + 2.0 ** -4 * ry.abs() * (1 + 1e-5) + 2.0 ** -10 * step).all())
    assert fb.int8_status() == 0


@pytest.mark.gpu
def test_layer_captured_and_replayed():
    """The whole layer in a graph on a side stream, replayed with other inputs: the bits of an eager
    call; and two graphs of it replayed at the same time."""
    graphs = []
    for seed, T in ((1, 40), (2, 200)):
        args = _layer_inputs(T, 512, 256, 32, seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _layer(*args, 0)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = _layer(*args, 0)
        graphs.append((graph, s, args, got, T))
    for round_ in range(3):
        for _, _, args, _, T in graphs:
            new = _layer_inputs(T, 512, 256, 32, 10 + round_)
            for old, n in zip(args[:7], new[:7]):
                old.copy_(n)
        torch.cuda.synchronize()
        for graph, s, *_ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, args, got, _ in graphs:
            want = _layer(*args, 0)
            for k in ("hidden", "up", "down", "y", "out"):
                assert torch.equal(got[k], want[k]), k
            assert torch.equal(got["q8"][0].view(torch.uint8), want["q8"][0].view(torch.uint8))


@pytest.mark.gpu
def test_layer_from_several_threads_at_once():
    """Four host threads, each on its own stream: the bits of one call after the other."""
    args = [_layer_inputs(T, 512, 256, 32, 30 + T) for T in (3, 40, 200, 64)]
    want = [_layer(*a, 0) for a in args]
    torch.cuda.synchronize()
    got = [None] * len(args)

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                r = _layer(*args[i], 0)
            s.synchronize()
        got[i] = r

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(args))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        for k in ("hidden", "up", "down", "y", "out"):
            assert torch.equal(g[k], w[k]), k
    assert fb.int8_status() == 0


@pytest.mark.gpu
def test_training_step_through_the_experts():
    """Norm, sort, one product per expert (torch), back with weights, norm: the gradients of every
    leaf against the same layer in 64 bits without any sorting."""
    T, H, E, K = 50, 64, 6, 3
    g = torch.Generator().manual_seed(0)

    def leaf(*shape, scale=1.0, base=0.0):
        return (base + scale * torch.randn(*shape, generator=g)).cuda().requires_grad_()
    x, w_pre, w_post = leaf(T, H), leaf(H, scale=0.1, base=1), leaf(H, scale=0.1, base=1)
    gate, W, weights = leaf(H), leaf(E, H, H, scale=0.1), leaf(T, K, scale=0.2, base=0.5)
    ids = torch.rand(T, E, generator=g).topk(K, 1).indices.int().cuda()
    up = torch.randn(T, H, generator=g).cuda()

    _, normed = fb.block_norm(None, x, pre_weight=w_pre)
    order = fb.sort_by_expert(ids, E)
    rows = fb.sort_tokens(normed, order)
    bases = order.expert_base.tolist()
    out = torch.cat([rows[a:b] @ W[e].t() for e, (a, b) in enumerate(zip(bases, bases[1:]))])
    y = fb.unsort_tokens(out, order, weights)
    h, _ = fb.block_norm(y, x, post_weight=w_post, gate=gate)
    leaves = [x, w_pre, w_post, gate, W, weights]
    got = torch.autograd.grad(h, leaves, up)

    d = [t.detach().double().requires_grad_() for t in leaves]
    n = d[0] / torch.sqrt(d[0].square().mean(1, keepdim=True) + 1e-6) * d[1]
    per = torch.einsum("th,tkgh->tkg", n, d[4][ids.long()])
    yy = (d[5][:, :, None] * per).sum(1)
    hh = d[0] + d[3] * (yy / torch.sqrt(yy.square().mean(1, keepdim=True) + 1e-6) * d[2])
    ref = torch.autograd.grad(hh, d, up.double())
    # fp32 throughout: sums of up to T * K * H = 9600 terms and a chain of four operators stay within
    # 2^-24 * (9600^0.5 * 40) of the largest gradient of each leaf, about 2.4e-4
    for a, b in zip(got, ref):
        assert float((a.double() - b).abs().max()) <= 2.4e-4 * float(b.abs().max())


@pytest.mark.gpu
def test_norm_feeds_the_fp8_expert_layer():
    """block_norm's e4m3 form as run's input, against the oracle on the same bytes."""
    from oracle import moe as omoe
    from oracle import routing as orouting
    T, E = 8, 8
    act = wl.make_activations(T, 3)
    act.routing_logits[:, :E] += 3.0
    w = wl.local_weights(E, 0)
    g = torch.Generator().manual_seed(1)
    f, x = (torch.randn(T, wl.HIDDEN, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    one = torch.ones(wl.HIDDEN, dtype=torch.bfloat16, device="cuda")
    _, (q, s) = fb.block_norm(f, x, post_weight=one, pre_weight=one, quantize=True)
    out = fb.run(act.routing_logits.cuda(), act.routing_bias.cuda(), q, s,
                 *(t.cuda() for t in w), 0, wl.RSF_DEFAULT)
    ids, rw = orouting.route(act.routing_logits.numpy(), act.routing_bias.float().numpy(),
                             wl.RSF_DEFAULT)
    active = sorted({int(e) for e in ids.reshape(-1) if 0 <= e < E})
    W1 = {e: w[0][e].view(torch.uint8).numpy() for e in active}
    W2 = {e: w[2][e].view(torch.uint8).numpy() for e in active}
    ref = omoe.moe_reference(q.view(torch.uint8).cpu().numpy(), s.cpu().numpy(), W1, w[1].numpy(),
                             W2, w[3].numpy(), ids, rw, 0)
    frac, err = omoe.allclose_report(out.view(torch.int16).cpu().numpy().view(np.uint16), ref,
                                     atol=1e-2, rtol=1e-2)
    assert frac == 1.0, err


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows, products and norms of more than 2^31 elements: the last ones are right."""
    bf = torch.bfloat16
    T, K, H = 38000, 8, 7168                      # 304000 rows, 2.18e9 elements
    ids = torch.arange(8, dtype=torch.int32, device="cuda").repeat(T, 1)
    o = fb.sort_by_expert(ids, 8)
    x = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(0),
                    device="cuda").to(bf)
    rows = fb.sort_tokens(x, o)
    assert torch.equal(rows[7 * T:], x) and torch.equal(rows[:T], x)
    y = fb.unsort_tokens(rows, o)
    assert torch.equal(y, x * 8)                  # sums of eight equal bf16 are exact
    odd = fb.sort_tokens(x[:, :7167].contiguous(), o)
    assert torch.equal(odd[7 * T:], x[:, :7167])
    del odd, y
    h, n = fb.block_norm(rows, rows, residual_scale=1.0, pre_weight=torch.ones(H, device="cuda"))
    part = rows[-300:].double()
    eh, ey, *_ = R.block_norm_bounds(part, part, None, None, torch.ones(H, device="cuda").double(),
                                     1.0, 1e-6)
    rh, ry = R.block_norm(part, part, None, None, torch.ones(H, device="cuda").double(), 1.0, 1e-6)
    R.check(h[-300:], rh, eh, "hidden")
    R.check(n[-300:], ry, ey, "normed")
    q, s = fb.quantize_int8(rows)
    assert torch.equal(q[-300:].double(), R.quantize(rows[-300:])[0])
    del h, n, rows
    w = torch.randint(-128, 128, (7200, 16), device="cuda", dtype=torch.int8)
    w_s = torch.rand(7200, device="cuda")
    a = q[:, :16].contiguous()
    out = fb.int8_matmul(a, w, s, w_s)            # 304000 x 7200 outputs
    ref, err = R.product(a[-300:], w, s[-300:], w_s)
    R.check(out[-300:], ref, err, "product")
