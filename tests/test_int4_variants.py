"""Every tensor-core variant of the 4-bit products -- tiles of 64, 128 and 256 tokens, K whole and in up
to eight parts -- on the same sizes, whatever the size would choose."""
import ctypes
import time

import pytest
import torch

import flashinfer_b200 as fb
from flashinfer_b200 import _lib, int4
from tests import layer_refs as R
from tests.test_int4 import _case, _expert_check, _gen, _product

VARIANTS = [(bn, s) for bn in (64, 128, 256) for s in (1, 2, 5, 8)]


@pytest.fixture
def variant(monkeypatch):
    """variant(bn, split): the next product takes it."""
    def arm(bn, split):
        assert _lib.load().fmoe_debug_arm_int4_plan(bn, split) == 0
        monkeypatch.setattr(int4, "_workspace_bytes",
                            lambda M, N, K, E: split * M * N * 4 if split > 1 else 0)
    return arm


# M, N, K, group: a few tokens, one past a tile, odd N, K that ends inside a block, many K blocks (the
# ring wraps several times), more tiles than run at a time (a CTA takes several, over both accumulators)
SIZES = [(5, 33, 544, 32), (33, 257, 2080, 64), (130, 384, 4096, 128), (255, 65, 1056, 256),
         (300, 1000, 7168, 128), (517, 2047, 1632, 32), (1100, 7200, 2080, 64), (70, 130, 512, 8192),
         (260, 128, 1120, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,group", SIZES)
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_matmul(variant, bn, split, M, N, K, group):
    g = _gen(M + N + K)
    for dtype, zero, f32 in (("bf16", False, False), ("fp16", True, False), ("bf16", True, True),
                             ("fp16", False, True)):
        x, packed, scale, z = _case(g, M, N, K, group, dtype, zero, f32)
        bias = torch.randn(N, generator=g, device="cuda") if zero else None
        ref, err = _product(x, packed, scale, z, group, bias)
        variant(bn, split)
        R.check(fb.int4_matmul(x, packed, scale, z, bias, group=group), ref, err, (dtype, zero, f32))
    # an output between other values: nothing beyond it is written
    flat = torch.full((M * N + 2,), 3.0, device="cuda", dtype=x.dtype)
    variant(bn, split)
    fb.int4_matmul(x, packed, scale, z, bias, group=group, output=flat[1:-1].view(M, N))
    R.check(flat[1:-1].view(M, N), ref, err, "view")
    assert float(flat[0]) == 3.0 and float(flat[-1]) == 3.0
    assert fb.int4_status() == 0


# N, K, group, first row, counts per expert, rows behind the last expert
GROUPS = [(130, 544, 32, 0, [0, 3, 0, 2], 0),
          (96, 2080, 64, 5, [0, 0, 50, 1, 0, 17, 0, 0], 32),
          (301, 1056, 128, 0, [257, 0, 600, 16, 127], 9),
          (2100, 4128, 128, 3, [2999, 1], 0),
          (200, 544, 64, 40, [0, 0, 0], 0),
          (100, 512, 128, 2, [5] * 64 + [0] * 100 + [9] * 40, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,group,lo,counts,tail", GROUPS)
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_expert_matmul(variant, bn, split, N, K, group, lo, counts, tail):
    g = _gen(len(counts) + N)
    base = torch.tensor([lo] + counts, device="cuda").cumsum(0).to(torch.int32)
    M, E = int(base[-1]) + tail, len(counts)
    x, packed, scale, z = _case(g, M, N, K, group, "bf16", True, False, E)
    variant(bn, split)
    y = fb.int4_expert_matmul(x, packed, scale, base, z, group=group)
    _expert_check(y, x, packed, scale, z, group, base)
    assert not bool(y[:lo].any()) and not bool(y[int(base[-1]):].any())
    out = torch.full((M, N), 3.0, dtype=x.dtype, device="cuda")
    variant(bn, split)
    fb.int4_expert_matmul(x, packed, scale, base, z, group=group, output=out)
    assert bool((out[:lo] == 3).all()) and bool((out[int(base[-1]):] == 3).all())
    assert torch.equal(out[lo:int(base[-1])], y[lo:int(base[-1])])
    assert fb.int4_status() == 0


# bases that step back, over 700 rows: every expert names all rows (five times the tiles that 700 rows
# have), and steps in the middle, at the end and out of range
STEPS = [[0, 700, 0, 700, 0, 700], [5, 300, 20, 450, 450, 440], [-3, 90, 9000, -1, 650, 600],
         [700, 600, 500, 400, 300, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("base", STEPS)
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_bases_that_step_back_give_every_row_one_expert(variant, bn, split, base):
    x, packed, scale, z = _case(_gen(base[1]), 700, 257, 544, 32, "fp16", True, False, 5)
    bases = torch.tensor(base, dtype=torch.int32, device="cuda")
    variant(bn, split)
    y = fb.int4_expert_matmul(x, packed, scale, bases, z, group=32)
    clean = _expert_check(y, x, packed, scale, z, 32, bases)
    assert not bool(y[:clean[0]].any()) and not bool(y[clean[-1]:].any())
    variant(bn, split)
    assert torch.equal(y, fb.int4_expert_matmul(x, packed, scale, bases, z, group=32))
    assert fb.int4_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bn,split", [(64, 1), (128, 2), (256, 3)])
def test_far_scales(variant, bn, split):
    """Scales of one row from fp16's smallest to its largest: the large ones decide the result."""
    g = _gen(bn)
    x, packed, _, z = _case(g, 90, 70, 512, 64, "fp16", True, False)
    for f32 in (False, True):
        p = torch.randint(-24, -6, (70, 8), generator=g, device="cuda")
        p[:20] = torch.randint(-24, -20, (20, 8), generator=g, device="cuda")
        scale = torch.ldexp(torch.ones(70, 8, device="cuda"), p).to(torch.float32 if f32 else torch.float16)
        variant(bn, split)
        R.check(fb.int4_matmul(x, packed, scale, z, group=64), *_product(x, packed, scale, z, 64), f32)
    scale = torch.full((70, 8), 0.0, device="cuda", dtype=torch.float16)
    scale[3:] = 60000.0
    x = x * 2.0 ** -20
    variant(bn, split)
    R.check(fb.int4_matmul(x, packed, scale, z, group=64), *_product(x, packed, scale, z, 64), "large")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bn,split", [(64, 1), (128, 2), (256, 1)])
def test_non_finite_scales_stay_in_their_channel(variant, bn, split, dtype):
    x, packed, scale, z = _case(_gen(1), 90, 70, 512, 64, dtype, True, False)
    scale[5, 3], scale[9, 0] = float("nan"), float("inf")
    variant(bn, split)
    y = fb.int4_matmul(x, packed, scale, z, group=64)
    rest = [i for i in range(70) if i not in (5, 9)]
    assert bool(torch.isnan(y[:, 5]).all()) and not bool(torch.isfinite(y[:, 9]).any())
    ref, err = _product(x, packed[rest], scale[rest], z[rest], 64)
    R.check(y[:, rest], ref, err, "others")


@pytest.mark.gpu
@pytest.mark.parametrize("bn,split", VARIANTS)
def test_a_wait_that_runs_out_ends_the_product(variant, bn, split):
    """A wait that nothing ends gives up after its 5 ms in every variant, the status says so once, and
    the next product of the same variant (which needs the same tensor memory) is right."""
    x, packed, scale, z = _case(_gen(bn + split), 300, 1000, 4096, 128, "bf16", True, False)
    variant(bn, split)
    fb.int4_matmul(x, packed, scale, z)
    assert fb.int4_status() == 0
    assert _lib.load().fmoe_debug_arm_int4_timeout(5_000_000) == 0
    variant(bn, split)
    t0 = time.perf_counter()
    fb.int4_matmul(x, packed, scale, z)
    assert fb.int4_status() == _lib.STATUS_TIMEOUT_INT4
    assert time.perf_counter() - t0 < 1.0
    assert fb.int4_status() == 0
    variant(bn, split)
    R.check(fb.int4_matmul(x, packed, scale, z), *_product(x, packed, scale, z, 128), "after")
    assert fb.int4_status() == 0


def test_refusals_of_a_variant():
    lib = _lib.load()
    for bad in ((0, 1), (32, 1), (256, 0), (256, 9), (-64, 1)):
        assert lib.fmoe_debug_arm_int4_plan(*bad) == -2
    assert lib.fmoe_debug_arm_int4_timeout(1) == -2
    assert lib.fmoe_int4_status(None, None) == -1
    a = _lib.FmoeInt4Args()
    a.num_rows, a.n, a.k, a.num_experts, a.group, a.dtype, a.scale_dtype = 4, 16, 192, 1, 32, 1, 1
    a.x, a.weight, a.scale, a.out = 1 << 20, 2 << 20, 3 << 20, 4 << 20
    assert lib.fmoe_debug_arm_int4_plan(64, 4) == 0
    # three K blocks for four parts; refused once, the next call is back to its own choice
    assert lib.fmoe_int4_matmul(ctypes.byref(a), None) == -2
    assert lib.fmoe_debug_arm_int4_plan(64, 2) == 0
    assert lib.fmoe_int4_matmul(ctypes.byref(a), None) == -5          # no workspace for two parts
    a.num_rows = 0
    assert lib.fmoe_debug_arm_int4_plan(64, 2) == 0
    assert lib.fmoe_int4_matmul(ctypes.byref(a), None) == 0           # used up
    a.num_rows, a.out = 4, 1 << 20
    assert lib.fmoe_int4_matmul(ctypes.byref(a), None) == -2          # the output over x


# M, N, K, group: blocks enough for four warps each, of 16 rows, 32 rows and two sets of eight tokens; depths
# of one block of 128, of less than a warp each and of several steps; the next depth has eight warps again
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K,group", [
    (1, 4801, 4064, 128), (5, 4777, 96, 32), (8, 4730, 1120, 64), (2, 18977, 544, 128), (7, 18931, 2080, 32),
    (12, 4801, 4096, 64), (16, 4720, 288, 384), (9, 9473, 4128, 128), (3, 18931, 4128, 64)])
def test_few_tokens_of_short_rows(M, N, K, group, dtype):
    g = _gen(M + N + K)
    for zero in (False, True):
        x, packed, scale, z = _case(g, M, N, K, group, dtype, zero, zero)
        bias = torch.randn(N, generator=g, device="cuda") if zero else None
        R.check(fb.int4_matmul(x, packed, scale, z, bias, group=group),
                *_product(x, packed, scale, z, group, bias), zero)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N,K,group", [(421, 1056, 128), (610, 224, 32), (100, 4096, 64), (421, 4128, 128)])
def test_experts_of_short_rows(N, K, group, dtype):
    """Experts without rows, with one, with more than a set of eight."""
    g = _gen(N + K)
    counts = [0, 1, 20, 3, 8, 9, 0, 7] * 6
    E, M = len(counts), sum(counts) + 11
    base = (torch.tensor([0] + counts, device="cuda").cumsum(0) + 4).to(torch.int32)
    for zero in (False, True):
        x, packed, scale, z = _case(g, M, N, K, group, dtype, zero, zero, E)
        y = fb.int4_expert_matmul(x, packed, scale, base, z, group=group)
        _expert_check(y, x, packed, scale, z, group, base)
        assert not bool(y[:4].any()) and not bool(y[4 + sum(counts):].any())
