"""Dense layers in 8 bits on the GPU: tlm_mx8_quant bit for bit, tlm_add_rmsnorm, tlm_gemm_mx8 and
tlm_gemm_mx8_swiglu within their roundings of oracle/ref.py (float64), and runs of them together.

Tolerances. A rounding to 16 bits is off by half a step, finfo.eps / 2 of the value; an 8-bit code by half a step of its
place. fp32 arithmetic of a norm: 2^-18 of the value (64 roundings of 2^-24 at most in a sum's tree and the products
behind it). A product's sums: 2^-13 of the sum of the magnitudes (the matrix core keeps at least 17 bits of every one of
up to 128 products below the largest, of 16 times the mean magnitude)."""
import numpy as np
import pytest
import torch

from oracle import ref
from test_mx8_oracle import CUTS, GATED_CUTS, GATED_PLANS, PLANS
from tilelang.jit.adapter.mi355x import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
SUM, ARITH = 2.0 ** -13, 2.0 ** -18


def _empty(rows, K, fill=0xEE):
    """Buffers that a call writes, filled so that what it leaves alone can be told."""
    return (torch.full((rows, K), fill, dtype=torch.uint8, device=DEV).view(E4M3),
            torch.full(ops.mx8_scales_shape(rows, K), fill, dtype=torch.uint8, device=DEV).view(E8M0))


def _bytes(t):
    return t.view(torch.uint8).cpu().numpy()


def _check_unused(scales, rows, K, fill=0xEE):
    s = _bytes(scales)
    used = ref.mx8_tile_ref(np.ones((rows, K // 32), np.uint8), np.zeros_like(s))
    assert (s[used == 0] == fill).all()


def _operand(codes, byte):
    """Codes and scale bytes [rows, K / 32] on the GPU; places that no block has are NaN."""
    tiled = np.full(ops.mx8_scales_shape(*codes.shape), 255, np.uint8)
    return (torch.from_numpy(codes).to(DEV).view(E4M3),
            torch.from_numpy(ref.mx8_tile_ref(byte, tiled)).to(DEV).view(E8M0))


def _random(rows, K, g, wide=1.0):
    x = torch.randn(rows, K, generator=g).double() * torch.exp(wide * torch.randn(rows, 1, generator=g).double())
    return ref.mx8_quantise_ref(x)


def _whole(rows, K, g):
    """Whole numbers -4 .. 4 with scales 1/2, 1 and 2: sums of up to 1024 of their products are exact."""
    v = torch.randint(-4, 5, (rows, K), generator=g).float()
    byte = torch.randint(126, 129, (rows, K // 32), generator=g).byte().numpy()
    return v.to(E4M3).view(torch.uint8).numpy(), byte


# ---- quantiser


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,K,gap", [(1, 32, 0), (3, 160, 0), (64, 128, 8), (65, 4096, 1000), (130, 2080, 0),
                                        (1, 14336, 0), (7, 4128, 32)])
def test_quant_bit_exact(dtype, rows, K, gap):
    g = torch.Generator().manual_seed(rows + K)
    x = torch.randn(rows, K + gap, generator=g) * torch.exp(2 * torch.randn(rows, K + gap, generator=g))
    x = x.to(dtype)
    codes, scales = _empty(rows, K)
    ops.mx8_quant(x.to(DEV)[:, :K], codes, scales)
    want, byte = ref.mx8_quantise_ref(x[:, :K])
    assert np.array_equal(_bytes(codes), want)
    assert np.array_equal(ref.mx8_untile_ref(_bytes(scales), rows, K), byte)
    _check_unused(scales, rows, K)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_quant_every_value(dtype):
    """Every 16-bit pattern as its block's largest, and below larger ones."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.zeros(2048, 32 * 64, dtype=dtype)
    v = x.view(-1, 32)
    v[:65536, 5] = bits
    v[65536:, 9] = bits
    top = bits.abs().nan_to_num(0, 0, 0).float()
    v[65536:, 30] = torch.ldexp(top, torch.arange(65536) % 19).to(dtype)
    codes, scales = _empty(*x.shape)
    ops.mx8_quant(x.to(DEV), codes, scales)
    want, byte = ref.mx8_quantise_ref(x)
    assert np.array_equal(_bytes(codes), want)
    assert np.array_equal(ref.mx8_untile_ref(_bytes(scales), *x.shape), byte)


def test_quant_fp32_edges():
    """Scales' borders to the last bit, the smallest and largest numbers, subnormals, infinities, NaN."""
    e = torch.arange(-126, 127).double()
    b = torch.ldexp(torch.tensor(1.75, dtype=torch.float64), e).float()
    m = torch.cat([b, torch.nextafter(b, torch.tensor(float("inf"))), torch.nextafter(b, torch.tensor(0.0)),
                   torch.tensor([1.4e-45, 1e-40, 1.1754944e-38, 3.4028235e38, float("inf"), float("nan"), -float("inf")])])
    x = torch.zeros(m.numel(), 64)
    x[:, 33] = m
    x[:, 34] = m / 3
    x[:, 2] = -m
    codes, scales = _empty(*x.shape)
    ops.mx8_quant(x.to(DEV), codes, scales)
    want, byte = ref.mx8_quantise_ref(x)
    assert np.array_equal(_bytes(codes), want)
    assert np.array_equal(ref.mx8_untile_ref(_bytes(scales), *x.shape), byte)


# ---- norm


def _check_mx(codes, scales, exact, slack):
    """8-bit values within half a step of exact plus slack; each scale is that of a value within slack of the largest."""
    rows, K = exact.shape
    byte = ref.mx8_untile_ref(_bytes(scales), rows, K)
    got = ref.mx8_values_ref(_bytes(codes), byte)
    bad = ~np.isfinite(exact).reshape(rows, -1, 32).all(-1)
    assert np.array_equal(byte == 255, bad)
    assert not _bytes(codes).reshape(rows, -1, 32)[bad].any()
    ok = ~np.repeat(bad, 32, -1)
    exact, slack = np.where(ok, exact, 0), np.where(ok, slack, 0)
    big, s32 = (np.abs(v).reshape(rows, -1, 32) for v in (exact, slack))
    lo = ref.mx8_scale_ref(np.maximum(big - s32, 0).max(-1))
    hi = ref.mx8_scale_ref((big + s32).max(-1))
    assert ((byte >= lo) & (byte <= hi))[~bad].all()
    unit = np.repeat(2.0 ** (np.where(bad, 127, byte).astype(float) - 127), 32, -1)
    place = np.floor(np.log2(np.maximum((np.abs(exact) + slack) / unit, 2.0 ** -6)))
    half = 2.0 ** (place - 4) * unit
    assert (np.abs(np.where(ok, got, 0) - exact) <= half + slack).all()


def _norm_case(x, residual, w, eps, y, mx):
    rows, cols = x.shape
    d = [None if t is None else t.to(DEV) for t in (x, residual, w)]
    out = None if residual is None else torch.empty_like(d[1])
    yy = torch.full_like(d[0], 7.0) if y else None
    codes, scales = _empty(rows, cols) if mx else (None, None)
    ops.add_rmsnorm(d[0], d[1], d[2], out, eps, yy, codes, scales)
    want_out, want = ref.add_rmsnorm_ref(x, residual, w, eps)
    if residual is not None:
        assert torch.equal(out.cpu(), want_out)
    slack = ARITH * np.abs(want)
    if y:
        eps16 = torch.finfo(x.dtype).eps / 2
        tiny = 2.0 ** -25 if x.dtype is F16 else 0  # half of fp16's subnormal step
        got = yy.double().cpu().numpy()
        assert (np.abs(got - want) <= eps16 * np.abs(want) * (1 + ARITH) + slack + tiny).all()
    if mx:
        _check_mx(codes, scales, want, slack)
        _check_unused(scales, rows, cols)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (64, 128), (65, 544), (17, 4096), (5, 4128), (130, 5120),
                                       (2, 8192), (3, 16384), (1, 32768)])
@pytest.mark.parametrize("kind", ["same", "wide", "none"])
def test_norm(dtype, rows, cols, kind):
    g = torch.Generator().manual_seed(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * (1 + 15 * (torch.rand(cols, generator=g) < 0.05))).to(dtype)
    r = None if kind == "none" else (3 * torch.randn(rows, cols, generator=g)).to(dtype if kind == "same" else F32)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(dtype)
    _norm_case(x, r, w, 1e-6, True, True)


@pytest.mark.parametrize("rows,cols", [(1, 8), (5, 24), (3, 1000), (33, 4104)])
def test_norm_16_bit_only(rows, cols):
    g = torch.Generator().manual_seed(cols)
    x, r = (torch.randn(rows, cols, generator=g).to(BF16) for _ in "xr")
    _norm_case(x, r, None, 1e-5, True, False)
    _norm_case(x, None, None, 0.0, True, False)


@pytest.mark.parametrize("cols", [64, 4096])
def test_norm_8_bit_only_no_weight(cols):
    g = torch.Generator().manual_seed(cols)
    x, r = (torch.randn(70, cols, generator=g).to(F16) for _ in "xr")
    _norm_case(x, r, None, 1e-6, False, True)


def test_norm_in_place_rows_and_shape():
    g = torch.Generator().manual_seed(3)
    x, r = (torch.randn(4, 9, 256, generator=g).to(BF16) for _ in "xr")
    w = torch.randn(256, generator=g).to(BF16)
    stream, y = r.to(DEV), torch.empty_like(x, device=DEV)
    codes, scales = _empty(36, 256)
    ret = ops.add_rmsnorm(x.to(DEV), stream, w.to(DEV), stream, 1e-6, y, codes, scales)
    assert ret[0] is stream and ret[1] is y and ret[2] is codes and ret[3] is scales
    out, want = ref.add_rmsnorm_ref(x, r, w, 1e-6)
    assert torch.equal(stream.cpu(), out)
    _check_mx(codes, scales, want.reshape(36, 256), ARITH * np.abs(want.reshape(36, 256)))


def test_norm_zero_and_nan_rows():
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(4)).to(BF16)
    x[1] = 0
    x[2, 40] = float("nan")
    y = torch.empty_like(x, device=DEV)
    codes, scales = _empty(4, 128)
    ops.add_rmsnorm(x.to(DEV), None, None, None, 1e-6, y, codes, scales)
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3]].float()).all()
    byte = ref.mx8_untile_ref(_bytes(scales), 4, 128)
    assert (byte[1] == 1).all() and (byte[2] == 255).all() and not _bytes(codes)[1:3].any()


def test_norm_more_rows_than_a_launch_has_threads():
    """2^26 rows and some of 64 threads each: a launch counts 2^32 threads along a side."""
    rows = (1 << 26) + 70
    x = torch.randn(rows, 32, dtype=BF16, device=DEV)
    y = torch.zeros_like(x)
    ops.add_rmsnorm(x, None, None, None, 1e-6, y)
    at = torch.tensor([0, 1, (1 << 20) - 1, 1 << 20, (1 << 26) - 1, 1 << 26, rows - 1], device=DEV)
    _, want = ref.add_rmsnorm_ref(x[at].cpu(), None, None, 1e-6)
    got = y[at].double().cpu().numpy()
    assert (np.abs(got - want) <= (2.0 ** -8 * (1 + ARITH) + ARITH) * np.abs(want)).all()
    assert bool((y[-100000:] != 0).any(1).all())


def test_quant_past_32_bits():
    """Codes past 2^31 and 2^32 bytes."""
    rows, K = 140000, 32768
    x = torch.zeros(rows, K, dtype=F16, device=DEV)
    at = [0, 65535, 65536, 70001, 131072, rows - 1]
    g = torch.Generator().manual_seed(8)
    some = torch.randn(len(at), K, generator=g).half()
    x[at] = some.to(DEV)
    codes, scales = _empty(rows, K)
    ops.mx8_quant(x, codes, scales)
    want, byte = ref.mx8_quantise_ref(some)
    r = torch.tensor(at, device=DEV)
    assert np.array_equal(codes.view(torch.uint8)[r].cpu().numpy(), want)
    got = scales.view(torch.uint8)[r // 64, :, :, r % 64].cpu().numpy().reshape(len(at), -1)
    assert np.array_equal(got, byte)


# ---- products

SIZES = [(1, 1, 32), (1, 5, 64), (2, 32, 96), (3, 100, 128), (7, 64, 160), (15, 250, 1056), (16, 256, 416), (17, 33, 256),
         (31, 515, 128), (33, 64, 4096), (37, 130, 1056), (64, 192, 512), (65, 300, 288), (100, 260, 640), (128, 128, 128),
         (129, 257, 1024), (200, 1000, 2080), (257, 513, 384), (300, 70, 4096), (513, 260, 96)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gemm_exact_sums(dtype, M, N, K):
    """Whole numbers: every place of operands and scales is seen, whatever the order of the sums."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = _whole(M, K, g), _whole(N, K, g)
    if K > 1024:  # only so many products that their sum stays exact
        for m in (a, b):
            m[0][:, 512:-512] = 0
    guard = torch.full((M + 2, N), 7.0, dtype=dtype, device=DEV)
    c = guard[1:-1]
    ops.gemm_mx8(*_operand(*a), *_operand(*b), c)
    want, _ = ref.gemm_mx8_ref(a, b)
    assert torch.equal(c.cpu(), torch.from_numpy(want).to(dtype))
    assert (guard[0] == 7).all() and (guard[-1] == 7).all()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_gemm_random(M, N, K):
    g = torch.Generator().manual_seed(M * N + K)
    a, b = _random(M, K, g), _random(N, K, g)
    want, mag = ref.gemm_mx8_ref(a, b)
    for dtype in (BF16, F16):
        c = torch.full((M, N), 7.0, dtype=dtype, device=DEV)
        assert ops.gemm_mx8(*_operand(*a), *_operand(*b), c) is c
        got = c.double().cpu().numpy()
        h = torch.finfo(dtype).eps / 2
        tiny = 2.0 ** -25 if dtype is F16 else 0
        fits = np.abs(want) * (1 + 2 * h) + SUM * mag < torch.finfo(dtype).max
        assert (np.abs(got - want) <= h * np.abs(want) + (1 + h) * SUM * mag + tiny)[fits].all()


def _device_values(m):
    """float64 values on the GPU of an 8-bit operand, for sizes that are slow on the host."""
    codes, scales = m
    b = scales.view(torch.uint8).permute(0, 3, 1, 2).flatten(2).flatten(0, 1)
    e = b[:codes.shape[0], :codes.shape[1] // 32].double() - 127
    return codes.double() * torch.ldexp(torch.ones_like(e), e).repeat_interleave(32, 1)


@pytest.mark.parametrize("case", PLANS + CUTS)
def test_gemm_every_tile(case):
    """Each tile, with K whole and split, on whole numbers: equal bits; a graph's replay, which never splits, as well."""
    M, N, K = case[:3]
    g = torch.Generator().manual_seed(M + N)
    a, b = _whole(M, K, g), _whole(N, K, g)
    if K > 1024:
        for m in (a, b):
            m[0][:, 500:-500] = 0
    a, b = _operand(*a), _operand(*b)
    c = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
    for _ in range(3):
        ops.gemm_mx8(*a, *b, c)
    want = torch.matmul(_device_values(a), _device_values(b).T.contiguous()).to(BF16)
    assert torch.equal(c, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    d = torch.full_like(c, 7.0)
    with torch.cuda.graph(graph, stream=s):
        ops.gemm_mx8(*a, *b, d)
    for _ in range(3):
        d.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d, want)


@pytest.mark.parametrize("case", GATED_PLANS + GATED_CUTS)
def test_gemm_swiglu_every_tile(case):
    M, N, K = case[:3]
    g = torch.Generator().manual_seed(M + N)
    a, gate, up = (_whole(r, K, g) for r in (M, N, N))
    for m in (a, gate, up):  # exact sums, gates of a few units
        m[0][:, 500:] = 0
        m[1][:] -= 2
    a, gate, up = _operand(*a), _operand(*gate), _operand(*up)
    codes, scales = _empty(M, N)
    for _ in range(3):
        ops.gemm_mx8_swiglu(*a, *gate, *up, codes, scales)
    x = _device_values(a)
    v, u = (torch.matmul(x, _device_values(m).T.contiguous()) for m in (gate, up))
    want = (u * v * torch.sigmoid(v)).cpu().numpy()
    _check_mx(codes, scales, want, ARITH * np.abs(want) + 2.0 ** -126)
    _check_unused(scales, M, N)


def test_gemm_scales_far_apart():
    """Scales from 2^-126 to 2^120 whose sums fit; one block has them all, the others 1."""
    g = torch.Generator().manual_seed(9)
    e = torch.tensor([-126, -100, -60, -10, 0, 30, 90, 120])
    a, b = _whole(16, 128, g), _whole(16, 128, g)
    for m in (a, b):
        m[1][:] = 127
    a[0][:, 32:] = 0
    a[1][:8, 0] = (e + 127).byte().numpy()
    b[1][:8, 0] = (127 - e).byte().numpy()
    c = torch.empty(16, 16, dtype=BF16, device=DEV)
    ops.gemm_mx8(*_operand(*a), *_operand(*b), c)
    want, _ = ref.gemm_mx8_ref(a, b)
    fits = np.abs(want) < 2.0 ** 127
    fits &= (np.abs(want) > 2.0 ** -120) | (want == 0)
    assert np.array_equal(c.double().cpu().numpy()[fits], torch.from_numpy(want).to(BF16).double().numpy()[fits])


def test_gemm_nan_stays_in_its_row_and_column():
    g = torch.Generator().manual_seed(10)
    a, b = _random(70, 256, g, 0), _random(90, 256, g, 0)
    a[1][65, 3] = 255
    b[0][77, 200] = 0x7F
    c = torch.empty(70, 90, dtype=BF16, device=DEV)
    ops.gemm_mx8(*_operand(*a), *_operand(*b), c)
    nan = torch.isnan(c).cpu()
    want = torch.zeros(70, 90, dtype=torch.bool)
    want[65] = want[:, 77] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("M,N", [(3, 40), (1000, 1024), (4096, 4096)])
def test_no_columns_of_k(M, N):
    """Sums of nothing: zeros, from every tile."""
    a, b = _empty(M, 0), _empty(N, 0)
    c = torch.full((M, N), 7.0, dtype=F16, device=DEV)
    ops.gemm_mx8(*a, *b, c)
    assert not c.any()
    if N % 32 == 0:
        codes, scales = _empty(M, N)
        ops.gemm_mx8_swiglu(*a, *b, *b, codes, scales)
        assert not codes.view(torch.uint8).any()
        assert (ref.mx8_untile_ref(_bytes(scales), M, N) == 1).all()


def test_gemm_past_32_bits():
    """Operands and a result past 2^31 bytes: the rows about the borders and the last ones."""
    g = torch.Generator().manual_seed(21)
    M, N, K = 600000, 2048, 4128
    a, b = _whole(64, K, g), _whole(N, K, g)
    for m in (a, b):
        m[0][:, 500:-500] = 0
    big = torch.zeros(M, K, dtype=torch.uint8, device=DEV)
    s = torch.full(ops.mx8_scales_shape(M, K), 127, dtype=torch.uint8, device=DEV)
    codes = torch.from_numpy(a[0]).to(DEV)
    at = [0, 64 * 8127, 64 * 8191, 64 * (M // 64 - 1)]  # whole groups of 64 rows
    for r in at:
        big[r:r + 64] = codes
        s[r // 64] = _operand(*a)[1].view(torch.uint8)[0]
    c = torch.full((M, N), 7.0, dtype=BF16, device=DEV)
    ops.gemm_mx8(big.view(E4M3), s.view(E8M0), *_operand(*b), c)
    want = torch.from_numpy(ref.gemm_mx8_ref(a, b)[0]).to(BF16).to(DEV)
    for r in at:
        assert torch.equal(c[r:r + 64], want)
    assert not c[64:64 * 8127].any() and not c[-64 - M % 64 - 1:-64 - M % 64].any()


@pytest.mark.parametrize("M", [5, 300])
def test_gemm_first_and_last_scale(M):
    """Scales that the quantiser never writes but others may: 2^-127 and 2^127, in products that fit."""
    g = torch.Generator().manual_seed(M)
    a, b = _whole(M, 256, g), _whole(64, 256, g)
    a[1][:], b[1][:] = 0, 254
    c = torch.empty(M, 64, dtype=BF16, device=DEV)
    ops.gemm_mx8(*_operand(*a), *_operand(*b), c)
    assert torch.equal(c.cpu(), torch.from_numpy(ref.gemm_mx8_ref(a, b)[0]).to(BF16))


@pytest.mark.parametrize("M,N,K", [(1, 32, 32), (2, 64, 160), (16, 96, 1056), (17, 128, 256), (33, 544, 128), (64, 256, 4096),
                                   (65, 64, 640), (100, 1056, 96), (128, 128, 1024), (130, 320, 512), (257, 288, 384),
                                   (300, 2048, 256)])
def test_gemm_swiglu(M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    a, gate, up = _random(M, K, g, 0.3), _random(N, K, g, 0.3), _random(N, K, g, 0.3)
    for m in (gate, up):
        m[1][:] -= int(np.log2(K) / 2)  # weights as a layer has them
    codes, scales = _empty(M, N)
    ret = ops.gemm_mx8_swiglu(*_operand(*a), *_operand(*gate), *_operand(*up), codes, scales)
    assert ret[0] is codes and ret[1] is scales
    want, move = ref.gemm_mx8_swiglu_ref(a, gate, up)
    _check_mx(codes, scales, want, SUM * 2 * move + ARITH * np.abs(want) + 2.0 ** -126)
    _check_unused(scales, M, N)


@pytest.mark.parametrize("M,N,K", [(1, 512, 4096), (13, 320, 2080), (32, 2048, 1024), (32, 64, 4096)])
def test_gemm_swiglu_few_rows(M, N, K):
    """Up to 32 rows are summed in fp32: K / 32 + 40 roundings of 2^-24 at most, below 2^-16 of the magnitudes."""
    g = torch.Generator().manual_seed(M * N)
    a, gate, up = _random(M, K, g, 0.3), _random(N, K, g, 0.3), _random(N, K, g, 0.3)
    for m in (gate, up):
        m[1][:] -= int(np.log2(K) / 2)
    codes, scales = _empty(M, N)
    ops.gemm_mx8_swiglu(*_operand(*a), *_operand(*gate), *_operand(*up), codes, scales)
    want, move = ref.gemm_mx8_swiglu_ref(a, gate, up)
    _check_mx(codes, scales, want, 2.0 ** -16 * move + ARITH * np.abs(want) + 2.0 ** -126)
    _check_unused(scales, M, N)


def test_gemm_swiglu_large_gates():
    """Gates of +-hundreds: exp overflows to infinity or vanishes, the result is up * gate or 0; NaN fills its block."""
    g = torch.Generator().manual_seed(12)
    a, gate, up = _whole(20, 64, g), _whole(64, 64, g), _whole(64, 64, g)
    gate[1][:] += 6
    a[1][7, 0] = 255
    codes, scales = _empty(20, 64)
    ops.gemm_mx8_swiglu(*_operand(*a), *_operand(*gate), *_operand(*up), codes, scales)
    want, move = ref.gemm_mx8_swiglu_ref(a, gate, up)
    want[np.abs(want) < 2.0 ** -126] = 0
    _check_mx(codes, scales, want, ARITH * np.abs(want) + 2.0 ** -126)


# ---- runs of them together


def _layer(M, hidden, inter, seed=0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    t = dict(x=torch.randn(M, hidden, generator=g).to(dtype), residual=torch.randn(M, hidden, generator=g).to(dtype),
             w=(1 + 0.1 * torch.randn(hidden, generator=g)).to(dtype))
    w = {n: (torch.randn(r, k, generator=g) / k ** 0.5).to(dtype)
         for n, r, k in (("o", hidden, hidden), ("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter))}
    return t, w


def _run_layer(d, q, bufs):
    """Attention's outputs x -> projection -> residual and norm -> gated block -> residual and norm."""
    ops.mx8_quant(d["x"], *bufs["x8"])
    ops.gemm_mx8(*bufs["x8"], *q["o"], bufs["c"])
    ops.add_rmsnorm(bufs["c"], d["residual"], d["w"], bufs["r"], 1e-6, None, *bufs["n8"])
    ops.gemm_mx8_swiglu(*bufs["n8"], *q["gate"], *q["up"], *bufs["h8"])
    ops.gemm_mx8(*bufs["h8"], *q["down"], bufs["c"])
    ops.add_rmsnorm(bufs["c"], bufs["r"], d["w"], bufs["r2"], 1e-6, bufs["y"])


def _buffers(M, hidden, inter, dtype=BF16):
    def e():
        return torch.empty(M, hidden, dtype=dtype, device=DEV)
    return dict(x8=_empty(M, hidden), n8=_empty(M, hidden), h8=_empty(M, inter), c=e(), r=e(), r2=e(), y=e())


def _quantised(w):
    q = {}
    for n, t in w.items():
        q[n] = _empty(*t.shape)
        ops.mx8_quant(t.to(DEV), *q[n])
    return q


@pytest.mark.parametrize("M,hidden,inter", [(1, 256, 736), (5, 512, 1408), (70, 288, 544), (200, 512, 1024)])
def test_layer(M, hidden, inter):
    t, w = _layer(M, hidden, inter)
    d, q, bufs = {k: v.to(DEV) for k, v in t.items()}, _quantised(w), _buffers(M, hidden, inter)
    _run_layer(d, q, bufs)
    # the same in float64 with the operators' own roundings between them
    v = {n: ref.mx8_values_ref(*ref.mx8_quantise_ref(m)) for n, m in w.items()}

    def mx(x):
        return ref.mx8_values_ref(*ref.mx8_quantise_ref(x))

    def r16(x):
        return torch.from_numpy(x).to(BF16)
    c = r16(mx(t["x"]) @ v["o"].T)
    r, n = ref.add_rmsnorm_ref(c, t["residual"], t["w"], 1e-6)
    a = mx(n)
    g, u = a @ v["gate"].T, a @ v["up"].T
    c = r16(mx(u * g / (1 + np.exp(-g))) @ v["down"].T)
    r2, y = ref.add_rmsnorm_ref(c, r, t["w"], 1e-6)
    # roundings that fall the other way are single steps of 8 or 16 bits: a small part of what eight of them make
    got = bufs["y"].double().cpu().numpy()
    assert np.linalg.norm(got - y) <= 8 * 2.0 ** -8 * np.linalg.norm(y)


def test_graph_replays():
    M, hidden, inter = 9, 512, 1056
    t, w = _layer(M, hidden, inter, 1)
    d, q, bufs = {k: v.to(DEV) for k, v in t.items()}, _quantised(w), _buffers(M, hidden, inter)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run_layer(d, q, bufs)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        _run_layer(d, q, bufs)
    for seed in range(3):
        new, _ = _layer(M, hidden, inter, 10 + seed)
        for k, v in new.items():
            d[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        other = _buffers(M, hidden, inter)
        _run_layer(d, q, other)
        torch.cuda.synchronize()
        a, b = bufs["y"].double(), other["y"].double()
        assert (a - b).norm() <= 2.0 ** -6 * b.norm()


def test_two_streams_at_once():
    """Products that split K use the stream's own workspace."""
    M, hidden, inter = 40, 1024, 2048
    t, w = _layer(M, hidden, inter, 2)
    d, q = {k: v.to(DEV) for k, v in t.items()}, _quantised(w)
    want = _buffers(M, hidden, inter)
    _run_layer(d, q, want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    bufs = [_buffers(M, hidden, inter) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, b in zip(streams, bufs):
            with torch.cuda.stream(s):
                _run_layer(d, q, b)
    torch.cuda.synchronize()
    for b in bufs:
        assert torch.equal(b["y"], want["y"])


def test_same_bits_again():
    g = torch.Generator().manual_seed(5)
    for M, N, K in ((1, 4096, 4096), (16, 1000, 8192), (64, 4096, 7168), (300, 1024, 4096)):
        a, b = (_operand(*_random(r, K, g)) for r in (M, N))
        c = [torch.empty(M, N, dtype=BF16, device=DEV) for _ in range(4)]
        for x in c:
            ops.gemm_mx8(*a, *b, x)
        for x in c[1:]:
            assert torch.equal(x, c[0])
