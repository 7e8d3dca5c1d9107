"""Every tensor-core variant of the int8 products -- tiles of 16, 64 and 128 tokens, CTA pairs, each with
K whole and split in 2 to 4 -- on the same sizes, whatever the size would choose."""
import threading
import time

import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib
from tests import layer_refs as R

VARIANTS = [(bn, s) for bn in (16, 64, 128, 256) for s in (1, 2, 3, 4)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int8(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def _arm(bn, split):
    assert _lib.load().fmoe_debug_arm_int8_plan(bn, split) == 0


# M, N, K: a few tokens, one past a tile, odd N, K that ends inside a block, many K blocks (the ring
# wraps several times), more tiles than run at a time (a CTA takes several, over both accumulators)
SIZES = [(5, 33, 528), (33, 257, 2064), (130, 384, 4096), (255, 65, 1040), (300, 1000, 7168),
         (517, 2047, 1616), (1100, 7200, 2064)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_matmul(bn, split, M, N, K):
    g = _gen(M + N + K)
    a, w = _int8(g, M, K), _int8(g, N, K)
    a_s = torch.rand(M, generator=g, device="cuda") + 0.01
    w_s = torch.rand(N, generator=g, device="cuda") * 1e-6     # inside fp16's range
    bias = torch.randn(N, generator=g, device="cuda")
    for dtype, b in ((torch.bfloat16, None), (torch.float32, bias), (torch.float16, bias)):
        ref, err = R.product(a, w, a_s, w_s, b)
        _arm(bn, split)
        R.check(fb.int8_matmul(a, w, a_s, w_s, b, out_dtype=dtype), ref, err, str(dtype))
    # an output between other values: nothing beyond it is written
    flat = torch.full((M * N + 2,), 3.0, device="cuda", dtype=torch.bfloat16)
    _arm(bn, split)
    fb.int8_matmul(a, w, a_s, w_s, output=flat[1:-1].view(M, N))
    ref, err = R.product(a, w, a_s, w_s)
    R.check(flat[1:-1].view(M, N), ref, err, "view")
    assert float(flat[0]) == 3.0 and float(flat[-1]) == 3.0
    assert fb.int8_status() == 0


def test_no_group_of_a_tile_lies_beyond_its_shares():
    """The arithmetic of a split tile: its tokens in groups of 16 up to the last token, its shares of
    whole groups. Every group belongs to one of the S shares."""
    for rows in range(1, 257):
        for S in (2, 3, 4):
            per = -(-(-(-rows // S)) // 16) * 16
            assert all(c // per < S for c in range(0, rows, 16)), (rows, S)
    # while the MMA's columns, which pairs round up to 32, do have groups beyond: 144 of 160
    assert 144 // 48 == 3


@pytest.mark.gpu
@pytest.mark.parametrize("M", [33, 129, 130, 144, 300, 517])
def test_pairs_whose_columns_exceed_their_shares(M):
    N, K = 257, 1040
    g = _gen(M)
    a, w = _int8(g, M, K), _int8(g, N, K)
    a_s = torch.rand(M, generator=g, device="cuda") + 0.01
    w_s = torch.rand(N, generator=g, device="cuda")
    ref, err = R.product(a, w, a_s, w_s)
    _arm(256, 3)
    R.check(fb.int8_matmul(a, w, a_s, w_s, out_dtype=torch.float32), ref, err, "split in 3")
    assert fb.int8_status() == 0


# E, N, K, first row, counts per expert, rows behind the last expert
GROUPS = [(4, 130, 528, 0, [0, 3, 0, 2], 0),
          (8, 96, 2064, 5, [0, 0, 50, 1, 0, 17, 0, 0], 32),
          (5, 301, 1040, 0, [257, 0, 600, 16, 127], 9),
          (2, 2100, 4112, 3, [2999, 1], 0),
          (3, 200, 528, 40, [0, 0, 0], 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("E,N,K,lo,counts,tail", GROUPS)
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_expert_matmul(bn, split, E, N, K, lo, counts, tail):
    g = _gen(E + N)
    base = [lo]
    for c in counts:
        base.append(base[-1] + c)
    Rn = base[-1] + tail
    rows, w = _int8(g, Rn, K), _int8(g, E, N, K)
    r_s = torch.rand(Rn, generator=g, device="cuda") + 0.01
    w_s = torch.rand(E, N, generator=g, device="cuda") * 1e-3
    ref = torch.zeros(Rn, N, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(ref)
    for e in range(E):
        a, b = base[e], base[e + 1]
        ref[a:b], err[a:b] = R.product(rows[a:b], w[e], r_s[a:b], w_s[e])
    bases = torch.tensor(base, dtype=torch.int32, device="cuda")
    _arm(bn, split)
    R.check(fb.int8_expert_matmul(rows, w, r_s, w_s, bases), ref, err, "rows")
    out = torch.full((Rn, N), 3.0, device="cuda")
    _arm(bn, split)
    fb.int8_expert_matmul(rows, w, r_s, w_s, bases, output=out)
    ref[:lo] = 3.0
    ref[base[-1]:] = 3.0
    R.check(out, ref, err, "given output")
    assert fb.int8_status() == 0


# bases that step back, over 700 rows: every expert names all rows (five times the tiles that 700 rows
# have), and steps in the middle, at the end and out of range
STEPS = [[0, 700, 0, 700, 0, 700], [5, 300, 20, 450, 450, 440], [-3, 90, 9000, -1, 650, 600],
         [700, 600, 500, 400, 300, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("base", STEPS)
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_bases_that_step_back_give_every_row_one_expert(bn, split, base):
    Rn, E, N, K = 700, 5, 257, 528
    g = _gen(base[1])
    rows, w = _int8(g, Rn, K), _int8(g, E, N, K)
    r_s = torch.rand(Rn, generator=g, device="cuda") + 0.01
    w_s = torch.rand(E, N, generator=g, device="cuda")
    up, most = [], 0
    for b in base:
        most = max(most, min(max(b, 0), Rn))
        up.append(most)
    ref = torch.zeros(Rn, N, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(ref)
    for e in range(E):
        a, b = up[e], up[e + 1]
        ref[a:b], err[a:b] = R.product(rows[a:b], w[e], r_s[a:b], w_s[e])
    bases = torch.tensor(base, dtype=torch.int32, device="cuda")
    _arm(bn, split)
    y = fb.int8_expert_matmul(rows, w, r_s, w_s, bases, out_dtype=torch.float32)
    R.check(y, ref, err, "rows")
    _arm(bn, split)
    assert torch.equal(y, fb.int8_expert_matmul(rows, w, r_s, w_s, bases, out_dtype=torch.float32))
    assert fb.int8_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_a_wait_that_runs_out_ends_the_product(bn, split):
    """A wait that nothing ends gives up after its 5 ms in every variant, the status says so once, and
    the next product of the same variant (which needs the same tensor memory) is right. In a CTA pair
    the injected failure also leaves one stage that only the leader has filled and one that only the
    other CTA has: waiting for copies that were never issued would take 2 s."""
    M, N, K = 300, 1000, 4096
    g = _gen(bn + split)
    a, w = _int8(g, M, K), _int8(g, N, K)
    a_s, w_s = torch.rand(M, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    _arm(bn, split)
    fb.int8_matmul(a, w, a_s, w_s)
    assert fb.int8_status() == 0
    assert _lib.load().fmoe_debug_arm_int8_timeout(5_000_000) == 0
    _arm(bn, split)
    t0 = time.perf_counter()
    fb.int8_matmul(a, w, a_s, w_s)
    assert fb.int8_status() == _lib.STATUS_TIMEOUT_INT8
    assert time.perf_counter() - t0 < 1.0
    assert fb.int8_status() == 0
    _arm(bn, split)
    y = fb.int8_matmul(a, w, a_s, w_s)
    ref, err = R.product(a, w, a_s, w_s)
    R.check(y, ref, err, "after")
    assert fb.int8_status() == 0


@pytest.mark.gpu
def test_no_failure_is_lost_to_a_concurrent_status_call():
    """A thread asks for the status without pause while products fail on another stream: each failure is
    seen by a call that ends after it."""
    M, N, K = 16, 128, 256
    g = _gen(0)
    a, w = _int8(g, M, K), _int8(g, N, K)
    a_s, w_s = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    fb.int8_matmul(a, w, a_s, w_s)
    assert fb.int8_status() == 0
    torch.cuda.synchronize()
    state = {"polls": 0, "seen": 0, "stop": False}

    def poll():
        with torch.cuda.stream(torch.cuda.Stream()):
            while not state["stop"]:
                if fb.int8_status():
                    state["seen"] += 1
                state["polls"] += 1

    t = threading.Thread(target=poll)
    t.start()
    lost = 0
    try:
        for _ in range(400):
            before = state["seen"]
            assert _lib.load().fmoe_debug_arm_int8_timeout(100_000) == 0
            fb.int8_matmul(a, w, a_s, w_s)
            torch.cuda.current_stream().synchronize()
            polls = state["polls"]
            end = time.perf_counter() + 5
            while state["polls"] < polls + 2 and time.perf_counter() < end:
                time.sleep(0)
            lost += state["seen"] == before
    finally:
        state["stop"] = True
        t.join()
    assert lost == 0
    assert fb.int8_status() == 0


def test_refusals_of_a_variant():
    lib = _lib.load()
    for bad in ((0, 1), (32, 1), (256, 0), (256, 5), (-16, 1)):
        assert lib.fmoe_debug_arm_int8_plan(*bad) == -2
    A, B, S, W, O = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
    assert lib.fmoe_debug_arm_int8_plan(64, 4) == 0
    # three K blocks for four parts; refused once, the next call is back to its own choice
    assert lib.fmoe_int8_matmul(A, B, S, W, None, 4, 8, 384, O, 1, None) == -2
    assert lib.fmoe_debug_arm_int8_plan(16, 2) == 0
    assert lib.fmoe_int8_matmul(A, B, S, W, None, 0, 8, 32, O, 1, None) == 0     # used up
    assert lib.fmoe_int8_matmul(A, B, S, W, None, 4, 8, 32, A + 64, 1, None) == -2
