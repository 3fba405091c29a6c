"""The tiles that 8-bit products take, without a GPU: what tlm_gemm_mx8_plan answers."""
import ctypes
import math
import random

import pytest

from test_mx8_oracle import EINVAL, EUNSUPPORTED, GATED_PLANS, PLANS, _refused, plan
from tilelang.jit.adapter.mi355x import lib

# gated products of few rows and more than 32768 columns, some whole rounds of 256 x 256 tiles and a rest: (M, N, K)
WIDE_COLUMNS = [(1, 33024, 512), (16, 33024, 4096), (1, 40960, 4096), (32, 40960, 256), (16, 53248, 16384), (32, 53248, 16384),
                (1, 65568, 8192), (32, 65568, 8192)]


@pytest.mark.parametrize("M,N,K", WIDE_COLUMNS)
def test_few_rows_of_many_columns_are_whole(M, N, K):
    """Up to 32 rows are summed in fp32, by tiles of 16 or 32 rows: no part of them goes to 256 x 256 tiles."""
    for split in (True, False):
        rows, cols, ns, first_rows, first_cols = plan(M, N, K, True, split)
        assert rows in (16, 32) and cols in (64, 128) and ns == 1
        assert (first_rows, first_cols) == (M, N)


# tlm_gemm_mx8_plan's `gated`
GATED, FP32_SUMS = 1, 2
# products that are summed in fp32, by every tile with K whole and, where calls take it so, split: (M, N, K, gated and fp32_sums,
# rows, columns of weights, whether workgroups share K). Gated ones of up to 32 rows are without being asked.
FP32_PLANS = [(1, 32, 4128, 1, 16, 64, True), (5, 1600, 544, 1, 16, 64, False), (20, 992, 32, 1, 16, 128, False),
              (5, 5024, 8192, 1, 16, 128, True), (17, 5024, 2080, 1, 32, 64, False), (17, 1600, 8192, 1, 32, 64, True),
              (30, 12000, 160, 1, 32, 128, False), (30, 5024, 14336, 1, 32, 128, True),
              (33, 32, 544, 3, 16, 64, False), (50, 96, 8192, 3, 16, 64, True), (50, 480, 96, 3, 16, 128, False),
              (130, 992, 4128, 3, 32, 64, False), (100, 480, 8192, 3, 32, 64, True), (100, 4096, 160, 3, 32, 128, False),
              (130, 992, 14336, 3, 32, 128, True), (130, 4096, 544, 3, 64, 128, False), (50, 5024, 8192, 3, 64, 128, True),
              (257, 12000, 96, 3, 128, 128, False), (100, 5024, 8192, 3, 128, 128, True),
              (1, 33, 544, 2, 16, 64, False), (1, 5003, 4128, 2, 16, 64, True), (400, 991, 1056, 2, 16, 128, False),
              (1, 9001, 8192, 2, 16, 128, True), (257, 1599, 2080, 2, 32, 64, False), (50, 1601, 8192, 2, 32, 64, True),
              (50, 8999, 32, 2, 32, 128, False), (20, 8999, 14336, 2, 32, 128, True), (257, 4095, 544, 2, 64, 128, False),
              (50, 8991, 8192, 2, 64, 128, True), (257, 8991, 160, 2, 128, 128, False), (400, 2559, 8192, 2, 128, 128, True)]


@pytest.mark.parametrize("case", FP32_PLANS)
def test_fp32_sums_plan(case):
    M, N, K, flags, rows, cols, split = case
    got = plan(M, N, K, flags)
    assert (*got[:2], got[2] > 1, *got[3:]) == (rows, cols, split, M, N)
    assert plan(M, N, K, flags, False)[2] == 1


@pytest.mark.parametrize("M", [1, 16, 17, 32, 33, 256, 4096])
def test_fp32_sums_take_no_8_bit_tile(M):
    """No tile of 16 or 32 columns, none of 256 x 256 and no part of them."""
    for N in (32, 480, 4096, 33024):
        for K in (0, 32, 4096, 14336):
            for flags in (FP32_SUMS, FP32_SUMS | GATED):
                rows, cols, _, *first = plan(M, N, K, flags)
                assert rows <= 128 and cols in (64, 128) and first == [M, N]
            # gated calls of few rows take the same without being asked
            assert M > 32 or plan(M, N, K, GATED) == plan(M, N, K, GATED | FP32_SUMS)


def test_fp32_sums_refusals():
    """More tiles of 128 x 128 (gated 128 x 64) than a launch has."""
    P = 1 << 20  # an address that is never read: these calls are refused first
    big = dict(M=1 << 20, N=(1 << 17) + 32, K=32)
    _refused("tlm_gemm_mx8_ex", P, P, P, P, P, *big.values(), lib.BF16, 1, None, code=EINVAL)
    _refused("tlm_gemm_mx8_swiglu_ex", P, P, P, P, P, P, P, P, *big.values(), 1, None, code=EINVAL)
    _refused("tlm_gemm_mx8_swiglu", P, P, P, P, P, P, P, P, *big.values(), None, code=EINVAL)
    with pytest.raises(lib.TLMError):
        plan(*big.values(), GATED | FP32_SUMS)
    assert plan(*big.values(), GATED)[0] == 256  # as 8-bit sums there is such a call
    assert plan(1 << 20, 1 << 15, 32, GATED | FP32_SUMS)[0] == 128
    # what the plain entry points refuse, these refuse as well
    _refused("tlm_gemm_mx8_ex", P, P, P, P, P, 4, 8, 48, lib.BF16, 1, None, code=EUNSUPPORTED)
    _refused("tlm_gemm_mx8_ex", P, P, P, P, P, 4, 8, 64, lib.F32, 1, None, code=EUNSUPPORTED)
    _refused("tlm_gemm_mx8_swiglu_ex", P, P, P, P, P, P, P, P, 4, 48, 64, 1, None, code=EUNSUPPORTED)
    _refused("tlm_gemm_mx8_swiglu_ex", P, None, P, P, P, P, P, P, 4, 64, 64, 1, None, code=EINVAL)


def test_plan_refuses_k_that_products_refuse():
    one, two = ctypes.c_int(), ctypes.c_int64()
    out = [ctypes.byref(one)] * 3 + [ctypes.byref(two)] * 2
    f = lib.load().tlm_gemm_mx8_plan
    for K in (2 ** 22 + 32, 2 ** 62, 2 ** 63 - 1):
        for flags in range(4):
            assert f(16, 4096, K, flags, 1, *out) == EINVAL
    assert f(16, 4096, 2 ** 22, 0, 1, *out) == 0


# products whose workgroups share K: (M, N, K, tlm_gemm_mx8_plan's `gated`)
SPLITS = [(3, 100, 14336, 0), (17, 2563, 14336, 0), (257, 1000, 14336, 0), (100, 9000, 8192, 0), (33, 992, 14336, 1),
          (257, 992, 8192, 1), (1100, 512, 8192, 1), (17, 1600, 8192, 1), (30, 5024, 14336, 1), (50, 1601, 8192, 2),
          (130, 992, 14336, 3)]


def test_splits_are_split():
    """What the tests of shared workspaces run uses them."""
    for case in SPLITS:
        assert plan(*case)[2] > 1 and plan(*case)[3:] == case[:2], case
        assert plan(*case, False)[2] == 1


# what PLANS and GATED_PLANS, whose gated products of 16-row tiles have up to 32 rows, leave out: (M, N, K, rows, columns of weights,
# whether workgroups share K), and gated
MORE_PLANS = [(2274, 61, 15552, 32, 64, True)]
MORE_GATED_PLANS = [(134, 64, 3712, 16, 64, False), (76, 64, 8224, 16, 64, True), (55, 2944, 352, 16, 128, False)]


@pytest.mark.parametrize("gated,case", [(0, c) for c in MORE_PLANS] + [(1, c) for c in MORE_GATED_PLANS])
def test_more_plans(gated, case):
    M, N, K, rows, cols, split = case
    got = plan(M, N, K, gated)
    assert (*got[:2], got[2] > 1, *got[3:]) == (rows, cols, split, M, N)


def _kernel(M, N, K, flags):
    """What tells kernels apart: gated, widened operands, tile, split."""
    rows, cols, ns, *_ = plan(M, N, K, flags)
    return flags & 1, bool(flags & FP32_SUMS or (flags & GATED and M <= 32)), rows, cols, ns > 1


def test_every_kernel_has_a_case():
    """No size takes a kernel that no GPU test of tiles takes."""
    tested = {_kernel(*c[:3], 0) for c in PLANS + MORE_PLANS} | {_kernel(*c[:3], 1) for c in GATED_PLANS + MORE_GATED_PLANS}
    tested |= {_kernel(*c[:4]) for c in FP32_PLANS}
    rng, taken = random.Random(0), {}
    for i in range(40000):
        M, N, K = (int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) for lo, hi in ((1, 8192), (1, 2000), (1, 512)))
        flags = i % 4
        N = 32 * N if flags & GATED else N * 32 - rng.randrange(32)
        taken.setdefault(_kernel(M, N, 32 * K, flags), (M, N, 32 * K, flags))
    assert not {k: v for k, v in taken.items() if k not in tested}
