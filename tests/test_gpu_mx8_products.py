"""Products of 8-bit operands on the GPU where a variant begins or ends: every tile on operands of any value, sums that the
matrix core cuts, blocks without a number, splits side by side. Tolerances are those of test_gpu_mx8.py."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import ref
from test_mx8_oracle import CUTS, GATED_CUTS, GATED_PLANS, PLANS, plan
from test_mx8_plans import FP32_PLANS, FP32_SUMS, MORE_GATED_PLANS, MORE_PLANS, SPLITS
from test_gpu_mx8 import ARITH, BF16, DEV, E4M3, E8M0, F16, SUM, _bytes, _check_mx, _check_unused, _device_values, _empty
from tilelang.jit.adapter.mi355x import ops

pytestmark = pytest.mark.gpu
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tilelang-tpu_amd")


def _rows(rows, K, g, scale=1.0):
    """Random rows, quantised."""
    x = scale * torch.randn(rows, K, generator=g, device=DEV) * torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEV))
    return ops.mx8_quant(x, *_empty(rows, K, 255))  # places that no block has are NaN


def _gated(a, gate, up):
    """up * silu(gate) in float64, and how far it moves when every product's magnitude is off by one part."""
    x, v, u = (_device_values(m) for m in (a, gate, up))
    v, u = v.T.contiguous(), u.T.contiguous()
    g, h = x @ v, x @ u
    gs, hs = x.abs() @ v.abs(), x.abs() @ u.abs()
    silu = g * torch.sigmoid(g)
    return (h * silu).cpu().numpy(), (silu.abs() * hs + 1.1 * h.abs() * gs).cpu().numpy()  # |silu'| < 1.1


def _fp32(K):
    """Of the products' magnitudes: a rounding of 2^-24 for every eight k, and 40 behind them."""
    return (K / 8 + 40) * 2.0 ** -24


@pytest.mark.parametrize("M,N,K", [(1, 33024, 512), (16, 33024, 288), (32, 40960, 256)])
def test_few_rows_of_many_columns(M, N, K):
    """Up to 32 rows are summed in fp32 whatever the columns, also where fp32_sums is False."""
    g = torch.Generator(device=DEV).manual_seed(N + M)
    a, gate, up = _rows(M, K, g), _rows(N, K, g, K ** -0.5), _rows(N, K, g, K ** -0.5)
    codes, scales = _empty(M, N)
    ops.gemm_mx8_swiglu(*a, *gate, *up, codes, scales, fp32_sums=False)
    want, move = _gated(a, gate, up)
    _check_mx(codes, scales, want, _fp32(K) * move + ARITH * np.abs(want) + 2.0 ** -126)
    _check_unused(scales, M, N)


def _cut_by_the_core(rows, K):
    """Rows whose products with themselves sum to 7, 2^14 + 7 - 2^14: the seven ones share a group of eight with the first
    2^14 and are below what the 8-bit instruction keeps beside it. fp32 sums hold them."""
    v = torch.zeros(rows, K)
    v[:, 0], v[:, 8], v[:, 1:8] = 128, -128, 1
    w = v.clone()
    w[:, 8] = 128

    def operand(x):
        s = torch.full(ops.mx8_scales_shape(rows, K), 127, dtype=torch.uint8, device=DEV)
        return x.to(DEV).to(E4M3), s.view(E8M0)
    return operand(v), operand(w)


@pytest.mark.parametrize("M,N,K", [(4112, 2048, 512), (4097, 2048, 4096), (4128, 4096, 256)])
def test_rows_of_one_call_are_summed_alike(M, N, K):
    """A rest of up to 32 rows behind whole rounds of 256 x 256 tiles: equal rows, equal results."""
    assert plan(M, N, K, True) == (256, 256, 1, 4096, N)
    a, w = _cut_by_the_core(M, K)[0], _cut_by_the_core(N, K)[1]
    codes, scales = _empty(M, N)
    ops.gemm_mx8_swiglu(*a, *w, *w, codes, scales, fp32_sums=False)
    c = codes.view(torch.uint8)
    assert torch.equal(c, c[:1].expand_as(c))
    s = scales.view(torch.uint8).permute(0, 3, 1, 2).flatten(2).flatten(0, 1)[:M]
    assert torch.equal(s, s[:1].expand_as(s))


@pytest.mark.parametrize("M,N,K", [(1, 64, 512), (17, 992, 4096), (33, 96, 8192), (300, 992, 512), (4112, 2048, 512)])
def test_fp32_sums_hold_what_cancels(M, N, K):
    """Sums of 7 = 2^14 + 7 - 2^14, whatever the tile: exact in fp32."""
    a, w = _cut_by_the_core(M, K)[0], _cut_by_the_core(N, K)[1]
    for dtype in (BF16, F16):
        c = torch.empty(M, N, dtype=dtype, device=DEV)
        assert ops.gemm_mx8(*a, *w, c, fp32_sums=True) is c
        assert bool((c == 7).all())
    codes, scales = _empty(M, N)
    ops.gemm_mx8_swiglu(*a, *w, *w, codes, scales)  # without being asked
    want = np.full((M, N), 49 / (1 + np.exp(-7.0)))
    _check_mx(codes, scales, want, ARITH * want)
    _check_unused(scales, M, N)


@pytest.mark.parametrize("case", FP32_PLANS)
def test_fp32_sums_every_tile(case):
    """Random operands within a bound on fp32's roundings; a graph's replay, which never splits, as well."""
    M, N, K, flags = case[:4]
    fp32_sums = bool(flags & FP32_SUMS)
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    a, b, up = _rows(M, K, g), _rows(N, K, g, K ** -0.5), _rows(N, K, g, K ** -0.5)
    if flags & 1:
        want, move = _gated(a, b, up)

        def check(codes, scales):
            _check_mx(codes, scales, want, _fp32(K) * move + ARITH * np.abs(want) + 2.0 ** -126)
            _check_unused(scales, M, N)

        def new():
            return _empty(M, N)

        def call(codes, scales):
            ops.gemm_mx8_swiglu(*a, *b, *up, codes, scales, fp32_sums=fp32_sums)
    else:
        x, y = _device_values(a), _device_values(b).T.contiguous()
        want, mag = x @ y, x.abs() @ y.abs()

        def check(c):
            h = 2.0 ** -8
            assert bool(((c.double() - want).abs() <= h * want.abs() + (1 + h) * _fp32(K) * mag).all())

        def new():
            return (torch.full((M, N), 7.0, dtype=BF16, device=DEV),)

        def call(c):
            ops.gemm_mx8(*a, *b, c, fp32_sums=True)
    for _ in range(3):
        out = new()
        call(*out)
        check(*out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph, out = torch.cuda.CUDAGraph(), new()
    with torch.cuda.graph(graph, stream=s):
        call(*out)
    for _ in range(3):
        for o in out:
            o.view(torch.uint8).fill_(0xEE)
        graph.replay()
        torch.cuda.synchronize()
        check(*out)


def _any(rows, K, g):
    """Codes of any finite value, so that products lie far apart, and scales of 2^-7 .. 2^7."""
    codes = torch.randint(0, 256, (rows, K), generator=g, device=DEV, dtype=torch.int32)
    codes = torch.where(codes % 128 == 127, codes - 1, codes).to(torch.uint8)
    scales = torch.randint(120, 135, ops.mx8_scales_shape(rows, K), generator=g, device=DEV, dtype=torch.int32)
    return codes.view(E4M3), scales.to(torch.uint8).view(E8M0)


def _powers(m):
    """2^exponent of every element as the matrix core takes it: a code below the least normal one has that one's."""
    codes, _ = m
    scale = _device_values((torch.full_like(codes.view(torch.uint8), 0x38).view(E4M3), m[1]))  # of codes 1
    field = (codes.view(torch.uint8) >> 3 & 15).clamp(min=1).double()
    return torch.exp2(field - 7) * scale


@pytest.mark.parametrize("case", PLANS + MORE_PLANS)
def test_bound_of_the_core(case):
    """The 8-bit instruction's sums: each product is cut below 2^-13 of the largest power of its eight neighbours, towards
    zero, and fp32 rounds once for every eight k and 40 times behind them."""
    M, N, K = case[:3]
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    a, b = _any(M, K, g), _any(N, K, g)
    c = torch.empty(M, N, dtype=BF16, device=DEV)
    ops.gemm_mx8(*a, *b, c)
    r, n = (torch.unique(torch.linspace(0, e - 1, 40, device=DEV).long()) for e in (M, N))
    x, y = _device_values(a)[r], _device_values(b)[n]
    want, mag = x @ y.T.contiguous(), x.abs() @ y.abs().T.contiguous()
    px, py = (t.unflatten(1, (-1, 8)) for t in (_powers(a)[r], _powers(b)[n]))
    top = sum((px[:, None, i:i + 64] * py[None, :, i:i + 64]).amax(-1).sum(-1) for i in range(0, K // 8, 64))
    h = 2.0 ** -8
    off = 7 * 2.0 ** -13 * top + _fp32(K) * mag
    assert bool(((c[r][:, n].double() - want).abs() <= h * want.abs() + (1 + h) * off).all())


# A process of its own: a stream keeps the workspace that it once took, and there are four.
SPLIT_STREAMS = """
import torch
from tilelang.jit.adapter.mi355x import ops
SPLITS = %r
g = torch.Generator(device="cuda").manual_seed(6)

def empty(rows, K):
    return (torch.zeros(rows, K, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            torch.zeros(ops.mx8_scales_shape(rows, K), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))

def rows(n, K, scale=1.0):
    return ops.mx8_quant(scale * torch.randn(n, K, generator=g, device="cuda"), *empty(n, K))

def call(case, x, out):
    M, N, K, flags = case
    if flags & 1:
        ops.gemm_mx8_swiglu(*x[0], *x[1], *x[2], *out, fp32_sums=bool(flags & 2))
    else:
        ops.gemm_mx8(*x[0], *x[1], *out, fp32_sums=bool(flags & 2))

def out(case):
    M, N, K, flags = case
    return empty(M, N) if flags & 1 else (torch.zeros(M, N, dtype=torch.float16, device="cuda"),)

def same(a, b):
    return all(bool(torch.equal(s.view(torch.uint8), t.view(torch.uint8))) for s, t in zip(a, b))

ins = [[rows(c[0], c[2]), rows(c[1], c[2], c[2] ** -0.5), rows(c[1], c[2], c[2] ** -0.5)] for c in SPLITS]
torch.cuda.synchronize()
streams = [torch.cuda.Stream() for _ in range(6)]
assert len({s.cuda_stream for s in streams}) == 6

def run(stream):
    res = [out(c) for c in SPLITS]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for c, x, o in zip(SPLITS, ins, res):
            call(c, x, o)
    return res

alone = [run(s) for s in streams]  # the first four take the workspaces
torch.cuda.synchronize()
captured = [out(c) for c in SPLITS]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=streams[0]):
    for c, x, o in zip(SPLITS, ins, captured):
        call(c, x, o)
for _ in range(3):  # a captured call never splits
    graph.replay()
    torch.cuda.synchronize()
    print("REPLAY", [same(o, a) for o, a in zip(captured, alone[5])])
together = [[run(s) for s in streams] for _ in range(8)]
torch.cuda.synchronize()
print("AGAIN", [[same(o, a) for o, a in zip(r, alone[i])].count(False) for t in together for i, r in enumerate(t)])
print("SPLIT", [[same(o, a) for o, a in zip(alone[i], alone[0])] for i in range(1, 4)])
print("WHOLE", [[same(o, a) for o, a in zip(alone[i], alone[0]) if len(o) == 1] for i in range(4, 6)])

def values(m):
    codes, scales = m
    b = scales.view(torch.uint8).permute(0, 3, 1, 2).flatten(2).flatten(0, 1)[:codes.shape[0], :codes.shape[1] // 32]
    return codes.double() * torch.exp2(b.double() - 127).repeat_interleave(32, 1)

worst = 0.0
for n, (M, N, K, flags) in enumerate(SPLITS):
    x, w, u = (values(m) for m in ins[n])
    want = x @ w.T.contiguous()
    if flags & 1:
        want = x @ u.T.contiguous() * want * torch.sigmoid(want)
    for r in alone:
        got = values(r[n]) if flags & 1 else r[n][0].double()
        limit = 2.0 ** -4 if flags & 1 else 2.0 ** -11 + 2.0 ** -13
        worst = max(worst, ((got - want).norm() / want.norm() / limit).item())
print("WORST", worst <= 1.0)
"""


def test_splits_on_six_streams():
    """Products that split K, of any operands, on six streams side by side: four own a workspace each, the others run unsplit;
    every stream repeats its bits whatever runs beside it, the four give the same ones, and a captured call has the unsplit ones."""
    r = subprocess.run([sys.executable, "-c", SPLIT_STREAMS % (SPLITS,)], capture_output=True, text=True, timeout=110, cwd=PKG)
    assert r.returncode == 0, r.stderr[-2000:]
    n = len(SPLITS)
    said = dict(line.split(" ", 1) for line in r.stdout.splitlines() if line.split(" ", 1)[0].isupper())
    assert r.stdout.count(f"REPLAY {[True] * n}") == 3, r.stdout
    assert said["AGAIN"] == str([0] * 48) and said["SPLIT"] == str([[True] * n] * 3) and said["WORST"] == "True", r.stdout
    # The others ran unsplit: sums of fp32 in another order round otherwise somewhere. (Of the 8-bit instruction's sums few do: what it
    # leaves of eight products is a multiple of 2^-13 of the largest, 2^11 of fp32's steps and more, so most sums are exact.)
    assert SPLITS[-2] == (50, 1601, 8192, 2) and said["WHOLE"].count("False]") == 2, r.stdout


# every tile, whole and split, and every cut: (M, N, K, tlm_gemm_mx8_plan's `gated`)
EVERY = [(*c[:3], 0) for c in PLANS + MORE_PLANS + CUTS] + [(*c[:3], 1) for c in GATED_PLANS + MORE_GATED_PLANS + GATED_CUTS]


def _products(a, b, up):
    """want = a @ b.T, the sum of its magnitudes, and the same of up, in float64."""
    x, v, u = (_device_values(m) for m in (a, b, up))
    v, u = v.T.contiguous(), u.T.contiguous()
    return x @ v, x.abs() @ v.abs(), x @ u, x.abs() @ u.abs()


@pytest.mark.parametrize("case", EVERY)
def test_every_tile_random(case):
    """Operands of any value over the whole of K."""
    M, N, K, gated = case
    g = torch.Generator(device=DEV).manual_seed(M * 3 + N + K)
    a, b, up = _rows(M, K, g), _rows(N, K, g, K ** -0.5), _rows(N, K, g, K ** -0.5)
    if gated:
        codes, scales = _empty(M, N)
        ops.gemm_mx8_swiglu(*a, *b, *up, codes, scales, fp32_sums=False)
        want, move = _gated(a, b, up)
        _check_mx(codes, scales, want, SUM * 2 * move + ARITH * np.abs(want) + 2.0 ** -126)
        _check_unused(scales, M, N)
        return
    x, y = _device_values(a), _device_values(b).T.contiguous()
    want, mag = x @ y, x.abs() @ y.abs()
    for dtype in (BF16, F16):
        c = torch.full((M, N), 7.0, dtype=dtype, device=DEV)
        ops.gemm_mx8(*a, *b, c)
        h, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype is F16 else 0
        assert bool(((c.double() - want).abs() <= h * want.abs() + (1 + h) * SUM * mag + tiny).all())


def _sparse(rows, K, at, g):
    """Whole numbers -4 .. 4 at the places `at` of every row, zeros elsewhere; scales 1/2, 1 and 2."""
    v = torch.zeros(rows, K, device=DEV)
    v[:, at] = torch.randint(-4, 5, (rows, len(at)), generator=g, device=DEV).float()
    s = torch.randint(126, 129, ops.mx8_scales_shape(rows, K), generator=g, device=DEV, dtype=torch.int32)
    return v.to(E4M3), s.to(torch.uint8).view(E8M0)


@pytest.mark.parametrize("case", EVERY)
def test_every_tile_exact_over_k(case):
    """Sums of whole numbers that lie all over K, in every stage and split: exact, whatever their order."""
    M, N, K, gated = case
    g = torch.Generator(device=DEV).manual_seed(M + N * 3 + K)
    at = torch.randperm(K, generator=g, device=DEV)[:500]
    at[0] = K - 1
    a, b, up = (_sparse(r, K, at, g) for r in (M, N, N))
    if gated:
        for m in (b, up):  # gates of a few units
            m[1].view(torch.uint8).sub_(4)
    x, v, u = (_device_values(m) for m in (a, b, up))
    v, u = x @ v.T.contiguous(), x @ u.T.contiguous()
    for _ in range(2):
        if gated:
            codes, scales = _empty(M, N)
            ops.gemm_mx8_swiglu(*a, *b, *up, codes, scales, fp32_sums=False)
            want = (u * v * torch.sigmoid(v)).cpu().numpy()
            _check_mx(codes, scales, want, ARITH * np.abs(want) + 2.0 ** -126)
        else:
            c = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
            ops.gemm_mx8(*a, *b, c)
            assert torch.equal(c, v.to(BF16))


def _call(case, a, b, up):
    """The bytes of a call's result on the host: codes and scales [M, N / 32] of a gated one."""
    M, N, K, flags = case
    fp32_sums = bool(flags & FP32_SUMS)
    if not flags & 1:
        c = torch.full((M, N), 7.0, dtype=F16, device=DEV)
        return ops.gemm_mx8(*a, *b, c, fp32_sums=fp32_sums).cpu(), None
    codes, scales = ops.gemm_mx8_swiglu(*a, *b, *up, *_empty(M, N), fp32_sums=fp32_sums)
    return codes.view(torch.uint8).cpu(), torch.from_numpy(ref.mx8_untile_ref(_bytes(scales), M, N))


@pytest.mark.parametrize("case", EVERY + [c[:4] for c in FP32_PLANS])
def test_blocks_without_a_number(case):
    """Rows and weights with a NaN or an infinity, as the quantiser writes their blocks (scale 255, codes 0): NaN in every result
    they take part in, and the same bits as without them everywhere else."""
    M, N, K, flags = case
    g = torch.Generator(device=DEV).manual_seed(M + N + K + flags)

    def rows(n, scale, bad):
        x = scale * torch.randn(n, K, generator=g, device=DEV)
        good = ops.mx8_quant(x, *_empty(n, K, 255))
        for r, k, v in bad:
            x[r, k] = v
        return good, ops.mx8_quant(x, *_empty(n, K, 255))
    inf, nan = float("inf"), float("nan")
    a, a_bad = rows(M, 1.0, [(M - 1, K - 1, nan), (M // 2, K // 3, -inf)])
    b, b_bad = rows(N, K ** -0.5, [(N - 1, 0, inf), (N // 3, K - 32, nan)])
    up, up_bad = rows(N, K ** -0.5, [(N // 2, K // 2, nan)])
    row, col = torch.zeros(M, 1, dtype=torch.bool), torch.zeros(1, N, dtype=torch.bool)
    row[[M - 1, M // 2]] = True
    col[0, [N - 1, N // 3]] = True
    plain, scales = _call(case, a, b, up)
    for ops_in, want in (((a_bad, b, up), row.expand(M, N)), ((a, b_bad, up), col.expand(M, N))):
        got, byte = _call(case, *ops_in)
        if flags & 1:  # a block of 32 columns has one scale
            want = want.unflatten(1, (-1, 32)).any(-1)
            assert torch.equal(byte == 255, want) and not got.unflatten(1, (-1, 32))[want].any()
            assert torch.equal(byte[~want], scales[~want])
            want = want.repeat_interleave(32, 1)
        else:
            assert torch.equal(torch.isnan(got), want)
        assert torch.equal(got[~want], plain[~want])
    if flags & 1:
        got, byte = _call(case, a, b, up_bad)
        want = torch.zeros(M, N // 32, dtype=torch.bool)
        want[:, N // 2 // 32] = True
        assert torch.equal(byte == 255, want) and torch.equal(byte[~want], scales[~want])


@pytest.mark.parametrize("M,hidden,inter", [(40, 1024, 1408), (300, 512, 2048), (1000, 2048, 1024)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_block_is_as_exact_as_16_bits(M, hidden, inter, dtype):
    """A gated feed-forward block by its plain calls, against float64 with the same 8-bit intermediates. The root mean square of a
    rounding to 16 bits is at most h / sqrt(3) of the value; a tenth more for the sums."""
    g = torch.Generator(device=DEV).manual_seed(M)
    a, gate, up = _rows(M, hidden, g), _rows(inter, hidden, g, hidden ** -0.5), _rows(inter, hidden, g, hidden ** -0.5)
    down = _rows(hidden, inter, g, inter ** -0.5)
    h8 = ops.gemm_mx8_swiglu(*a, *gate, *up, *_empty(M, inter))
    c = ops.gemm_mx8(*h8, *down, torch.empty(M, hidden, dtype=dtype, device=DEV))
    want, _ = _gated(a, gate, up)
    exact = torch.from_numpy(ref.mx8_values_ref(*ref.mx8_quantise_ref(want))).to(DEV) @ _device_values(down).T.contiguous()
    h = torch.finfo(dtype).eps / 2
    assert ((c.double() - exact).norm() / exact.norm()).item() <= 1.1 * h / 3 ** 0.5


@pytest.mark.parametrize("fp32_sums", [True, False])
def test_gated_past_32_bits(fp32_sums):
    """Codes of the result past 2^31 bytes, more rows than tiles of one height count in 16 bits: rows about the border and the last."""
    M, N, K = 531000, 4128, 96
    g = torch.Generator(device=DEV).manual_seed(13)
    at = torch.arange(K, device=DEV)
    some, gate, up = (_sparse(r, K, at, g) for r in (64, N, N))
    a = torch.zeros(M, K, dtype=torch.uint8, device=DEV)
    s = torch.full(ops.mx8_scales_shape(M, K), 127, dtype=torch.uint8, device=DEV)
    groups = [0, 2 ** 31 // N // 64 - 1, 2 ** 31 // N // 64, 2 ** 31 // N // 64 + 1, M // 64 - 1]
    for n in groups:
        a[64 * n:64 * n + 64] = some[0].view(torch.uint8)
        s[n] = some[1].view(torch.uint8)[0]
    codes, scales = ops.gemm_mx8_swiglu(a.view(E4M3), s.view(E8M0), *gate, *up, *_empty(M, N), fp32_sums=fp32_sums)
    want, _ = _gated(some, gate, up)
    for n in groups:
        _check_mx(codes[64 * n:64 * n + 64], scales[n:n + 1], want, ARITH * np.abs(want) + 2.0 ** -126)
    assert not codes.view(torch.uint8)[64:64 * groups[1]].any() and not codes.view(torch.uint8)[64 * (M // 64):].any()


@pytest.mark.parametrize("M,N", [(1, 64), (40, 96), (300, 512)])
def test_longest_k(M, N):
    """K of 2^22, the longest, in both kinds of sums."""
    K = 2 ** 22
    g = torch.Generator(device=DEV).manual_seed(M)
    at = torch.randperm(K, generator=g, device=DEV)[:500]
    at[0] = K - 1
    a, b = _sparse(M, K, at, g), _sparse(N, K, at, g)
    keep = at // 32  # the blocks that hold a value

    def values(m):
        byte = m[1].view(torch.uint8).permute(0, 3, 1, 2).flatten(2).flatten(0, 1)[:m[0].shape[0]][:, keep]
        return m[0].view(torch.uint8)[:, at].view(E4M3).double() * torch.exp2(byte.double() - 127)
    want = values(a) @ values(b).T.contiguous()
    for fp32_sums in (False, True):
        c = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
        ops.gemm_mx8(*a, *b, c, fp32_sums=fp32_sums)
        assert torch.equal(c, want.to(BF16))


@pytest.mark.parametrize("fp32_sums", [True, False])
def test_empty_calls(fp32_sums):
    """No rows, no columns: nothing is done; no k: zeros."""
    for M, N, K in ((0, 64, 96), (33, 0, 96), (0, 0, 0), (33, 64, 0), (1, 32, 0)):
        a, b = _empty(M, K, 0), _empty(N, K, 0)
        c = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
        ops.gemm_mx8(*a, *b, c, fp32_sums=fp32_sums)
        assert not c.any()
        codes, scales = ops.gemm_mx8_swiglu(*a, *b, *b, *_empty(M, N), fp32_sums=fp32_sums)
        assert not codes.view(torch.uint8).any()
        assert (ref.mx8_untile_ref(_bytes(scales), M, N) == 1).all()
        ops.mx8_quant(torch.zeros(M, K, device=DEV), *a)
    x = torch.zeros(0, 64, dtype=BF16, device=DEV)
    ops.add_rmsnorm(x, x, None, x, 0.0, x, *_empty(0, 64))
