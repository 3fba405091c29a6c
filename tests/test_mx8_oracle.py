"""Dense layers in 8 bits without a GPU: the oracle against torch's own e4m3 and a search over all codes, the
scales' layout, and what the entry points refuse."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import ref
from tilelang.jit.adapter.mi355x import lib, ops

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EINVAL, EUNSUPPORTED = -1, -2


def test_table_is_torch_e4m3():
    t = torch.arange(127, dtype=torch.uint8).view(E4M3).double().numpy()
    assert np.array_equal(t, ref.MX8_VALUES)


def test_quantise_nearest_and_scale():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 96, generator=g).double() * torch.exp(8 * torch.randn(40, 1, generator=g).double())
    codes, byte = ref.mx8_quantise_ref(x)
    s = 2.0 ** (byte.astype(float) - 127)
    big = np.abs(x.numpy()).reshape(40, 3, 32).max(-1)
    assert (big <= 448 * s).all() and (big > 224 * s).all()
    y = x.numpy().reshape(40, 3, 32) / s[..., None]
    d = np.abs(np.abs(y)[..., None] - ref.MX8_VALUES)
    got = np.abs(ref.mx8_values_ref(codes, byte)).reshape(y.shape) / s[..., None]
    assert np.array_equal(np.abs(got - np.abs(y)), d.min(-1))
    with torch.no_grad():
        assert np.array_equal(codes, torch.from_numpy(y.reshape(40, 96)).float().to(E4M3).view(torch.uint8).numpy())


def test_quantise_edges():
    x = np.zeros((6, 32))
    x[0, 3] = 448 * 2.0 ** 5           # the border of a scale
    x[1, 3] = np.nextafter(448 * 2.0 ** 5, 1e9)
    x[2, 0] = 2.0 ** -140               # below the least scale's range
    x[3, 7], x[4, 7] = np.inf, np.nan
    x[5, :2] = 448, -17                 # a tie: 16 or 18
    codes, byte = ref.mx8_quantise_ref(x)
    assert byte[:, 0].tolist() == [132, 133, 1, 255, 255, 127]
    assert codes[0, 3] == 126 and codes[1, 3] == 118 and not codes[2:5].any()
    assert ref.mx8_values_ref(codes, byte)[5, 1] == -16
    assert np.isnan(ref.mx8_values_ref(codes, byte)[3:5]).all()


@pytest.mark.parametrize("rows,K", [(1, 32), (64, 128), (65, 160), (130, 4096 + 96)])
def test_tile_scales(rows, K):
    b = torch.randint(0, 256, (rows, K // 32), generator=torch.Generator().manual_seed(1)).byte()
    got = ops.mx8_tile_scales(b.view(E8M0))
    assert got.dtype is E8M0 and got.shape == ops.mx8_scales_shape(rows, K)
    got = got.view(torch.uint8).numpy()
    assert np.array_equal(got, ref.mx8_tile_ref(b.numpy(), np.zeros_like(got)))
    assert np.array_equal(ref.mx8_untile_ref(got, rows, K), b.numpy())


def test_norm_ref():
    x = torch.tensor([[3.0, 4.0]]).half()
    out, y = ref.add_rmsnorm_ref(x, torch.tensor([[1.0, -1.0]]), None, 0.0)
    assert out.dtype is torch.float32 and np.allclose(y, np.array([[4.0, 3.0]]) / np.sqrt(12.5))


# ---- the choice of tile

# sizes for every tile, with K whole and, where calls take it so, split: (M, N, K, rows, columns of weights, workgroups per K is > 1)
PLANS = [(1, 32, 1056, 16, 16, False), (3, 100, 14336, 16, 16, True), (3, 9001, 1056, 16, 64, False),
         (5, 5003, 14336, 16, 64, True), (9, 9000, 96, 16, 128, False), (5, 9000, 14336, 16, 128, True),
         (20, 2563, 1056, 32, 16, False), (20, 1057, 14336, 32, 16, True), (30, 5003, 2080, 32, 32, False),
         (17, 2563, 14336, 32, 32, True), (257, 1000, 2080, 32, 64, False), (50, 9000, 160, 32, 128, False),
         (257, 1000, 14336, 32, 128, True), (400, 9000, 32, 64, 128, False), (33, 9000, 8192, 64, 128, True),
         (200, 9000, 1056, 128, 128, False), (100, 9000, 8192, 128, 128, True), (2000, 4096, 96, 256, 256, False)]
GATED_PLANS = [(1, 32, 1056, 16, 64, False), (3, 96, 8192, 16, 64, True), (9, 4096, 96, 16, 128, False),
               (5, 8992, 14336, 16, 128, True), (2000, 96, 1056, 32, 64, False), (33, 992, 14336, 32, 64, True),
               (257, 992, 160, 32, 128, False), (130, 992, 14336, 32, 128, True), (130, 8992, 32, 64, 128, False),
               (257, 992, 8192, 64, 128, True), (100, 8992, 1056, 128, 128, False), (1100, 512, 8192, 128, 128, True),
               (400, 8992, 96, 256, 256, False)]


def plan(M, N, K, gated, split=True):
    out = [ctypes.c_int() for _ in range(3)] + [ctypes.c_int64() for _ in range(2)]
    lib.call("tlm_gemm_mx8_plan", M, N, K, gated, split, *(ctypes.byref(o) for o in out))
    return tuple(o.value for o in out)


@pytest.mark.parametrize("gated,case", [(0, c) for c in PLANS] + [(1, c) for c in GATED_PLANS])
def test_plan(gated, case):
    M, N, K, rows, cols, split = case
    got = plan(M, N, K, gated)
    assert (*got[:2], got[2] > 1, *got[3:]) == (rows, cols, split, M, N)
    assert plan(M, N, K, gated, False)[2] == 1
    tiles = -(-M // rows) * -(-N // (cols // 2 if gated else cols))
    if split:  # the workspace holds the partial tiles
        assert tiles <= 512 and tiles * got[2] * rows * cols * 4 <= 16 << 20 and got[2] <= -(-K // 128) // 2


# more than whole rounds of 256 x 256 tiles: (M, N, K, rows and columns of the part that is whole rounds)
CUTS = [(4400, 4096, 2080, 4096, 4096), (2000, 9000, 4096, 2000, 8192), (4100, 4100, 1056, 3840, 4100)]
GATED_CUTS = [(4400, 2048, 2080, 4096, 2048), (2000, 4512, 4096, 2000, 4096), (2100, 4352, 1056, 2100, 3584)]


@pytest.mark.parametrize("gated,case", [(0, c) for c in CUTS] + [(1, c) for c in GATED_CUTS])
def test_plan_cuts(gated, case):
    M, N, K, rows, cols = case
    assert plan(M, N, K, gated) == (256, 256, 1, rows, cols)


def test_plan_refusals():
    one, two = ctypes.c_int(), ctypes.c_int64()
    f, out = lib.load().tlm_gemm_mx8_plan, [ctypes.byref(one)] * 3 + [ctypes.byref(two)] * 2
    assert f(0, 1, 32, 0, 1, *out) == EINVAL
    assert f(1, 1, 32, 0, 1, None, *out[1:]) == EINVAL and f(1, 1, 32, 0, 1, *out[:4], None) == EINVAL
    assert f(2 ** 31 - 256, 2 ** 31 - 256, 32, 0, 1, *out) == EINVAL


# ---- refusals

P = 1 << 20  # an address that is never read: every call here is refused first


def _refused(fn, *args, code=None):
    rc = getattr(lib.load(), fn)(*args)
    assert rc < 0 and (code is None or rc == code), rc
    msg = lib.load().tlm_last_error().decode()
    assert fn in msg
    return msg




def test_c_codes():
    import re
    text = open(__file__.replace("tests/test_mx8_oracle.py", "include/tlmi355x.h")).read()
    m = dict(re.findall(r"(TLM_E\w+)\s*=?\s*\(?(-\d+)\)?", text))
    assert int(m["TLM_EINVAL"]) == EINVAL and int(m["TLM_EUNSUPPORTED"]) == EUNSUPPORTED


def test_quant_refusals():
    f = "tlm_mx8_quant"
    ok = dict(x=P, stride=64, dt=lib.BF16, codes=P, scales=P, rows=4, cols=64)

    def call(code, **kw):
        a = dict(ok, **kw)
        return _refused(f, *a.values(), None, code=code)
    call(EUNSUPPORTED, cols=48)
    call(EUNSUPPORTED, dt=lib.F8E4M3)
    call(EINVAL, stride=63)
    call(EINVAL, stride=-64)
    call(EINVAL, x=P + 8)
    call(EINVAL, codes=P + 8)
    call(EINVAL, scales=P + 2)
    for n in ("x", "codes", "scales"):
        call(EINVAL, **{n: None})
    call(EINVAL, rows=-1)
    call(EINVAL, rows=2 ** 31)
    call(EINVAL, cols=2 ** 22 + 32)
    for kw in (dict(rows=0), dict(cols=0)):
        a = dict(ok, x=None, codes=None, scales=None, **kw)
        assert lib.load().tlm_mx8_quant(*a.values(), None) == 0


def test_norm_refusals():
    f = "tlm_add_rmsnorm"
    ok = dict(x=P, residual=P, w=P, out=P, y=P, codes=P, scales=P, rows=4, cols=64, eps=1e-6, dt=lib.BF16,
              rdt=lib.F32)

    def call(code, **kw):
        return _refused(f, *dict(ok, **kw).values(), None, code=code)
    call(EUNSUPPORTED, cols=40)
    call(EUNSUPPORTED, cols=44, codes=None, scales=None)
    call(EUNSUPPORTED, cols=1 << 21)
    call(EUNSUPPORTED, dt=lib.F32)
    call(EUNSUPPORTED, rdt=lib.F16)
    call(EINVAL, eps=-1.0)
    call(EINVAL, eps=float("nan"))
    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(residual=None), dict(out=None),
               dict(y=None, codes=None, scales=None), dict(cols=0, codes=None, scales=None), dict(rows=-1)):
        call(EINVAL, **kw)
    for n in ("x", "residual", "w", "out", "y", "codes"):
        call(EINVAL, **{n: P + 8})
    assert getattr(lib.load(), f)(*dict(ok, rows=0).values(), None) == 0


def test_gemm_refusals():
    f = "tlm_gemm_mx8"
    ok = dict(a=P, sa=P, b=P, sb=P, c=P, M=4, N=8, K=64, dt=lib.BF16)

    def call(code, **kw):
        return _refused(f, *dict(ok, **kw).values(), None, code=code)
    for n in ("a", "sa", "b", "sb", "c"):
        call(EINVAL, **{n: None})
        call(EINVAL, **{n: P + 1})
    call(EUNSUPPORTED, K=48)
    call(EUNSUPPORTED, dt=lib.F32)
    call(EINVAL, M=-1)
    call(EINVAL, N=2 ** 31)
    call(EINVAL, M=2 ** 30, N=2 ** 20)
    call(EINVAL, K=2 ** 22 + 32)
    for kw in (dict(M=0), dict(N=0)):
        assert getattr(lib.load(), f)(*dict(ok, **kw).values(), None) == 0


def test_swiglu_refusals():
    f = "tlm_gemm_mx8_swiglu"
    ok = dict(a=P, sa=P, g=P, sg=P, u=P, su=P, c=P, sc=P, M=4, N=64, K=64)

    def call(code, **kw):
        return _refused(f, *dict(ok, **kw).values(), None, code=code)
    for n in ("a", "sa", "g", "sg", "u", "su", "c", "sc"):
        call(EINVAL, **{n: None})
        call(EINVAL, **{n: P + 1})
    call(EUNSUPPORTED, K=48)
    call(EUNSUPPORTED, N=48)
    call(EINVAL, M=-1)
    for kw in (dict(M=0), dict(N=0)):
        assert getattr(lib.load(), f)(*dict(ok, **kw).values(), None) == 0


def _mx(rows, K):
    return torch.zeros(rows, K, dtype=E4M3), torch.zeros(ops.mx8_scales_shape(rows, K), dtype=torch.uint8).view(E8M0)


def test_front_refusals():
    """The Python front's own checks come before it looks for a device; what passes them fails for having none."""
    x, (c, s) = torch.zeros(3, 64).half(), _mx(3, 64)
    with pytest.raises(ValueError, match="HIP device"):
        ops.mx8_quant(x, c, s)
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.mx8_quant(torch.zeros(64, 3).half().T, c, s)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        ops.mx8_quant(x, c.view(torch.uint8), s)
    with pytest.raises(ValueError, match="scales of"):
        ops.mx8_quant(x, c, s.view(torch.uint8))
    with pytest.raises(ValueError, match="scales of"):
        ops.mx8_quant(x, c, _mx(65, 64)[1])
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        ops.mx8_quant(x, _mx(4, 64)[0], s)
    n = torch.zeros(64).half()
    ops_args = (x, x.float(), n, x.float(), 1e-6)
    with pytest.raises(ValueError, match="HIP device"):
        ops.add_rmsnorm(*ops_args, y=x.clone())
    for bad in (dict(), dict(codes=c), dict(y=x.float()), dict(y=x[:, :32]), dict(codes=c, scales=_mx(3, 160)[1])):
        with pytest.raises(ValueError):
            ops.add_rmsnorm(*ops_args, **bad)
    with pytest.raises(ValueError, match="together"):
        ops.add_rmsnorm(x, x, n, None, 1e-6, x)
    with pytest.raises(ValueError, match="residual's dtype"):
        ops.add_rmsnorm(x, x, n, x.float(), 1e-6, x)
    with pytest.raises(ValueError, match="w must"):
        ops.add_rmsnorm(x, x, n.float(), x, 1e-6, x)
    b, sb = _mx(5, 64)
    with pytest.raises(ValueError, match="HIP device"):
        ops.gemm_mx8(c, s, b, sb, torch.zeros(3, 5).half())
    for args in ((c, s, *_mx(5, 96), torch.zeros(3, 5).half()), (c, s, b, sb, torch.zeros(5, 3).half()),
                 (c, s, b, sb, torch.zeros(5, 3).half().T), (c[0], s, b, sb, torch.zeros(3, 5).half())):
        with pytest.raises(ValueError):
            ops.gemm_mx8(*args)
    with pytest.raises(ValueError, match="B_up"):
        ops.gemm_mx8_swiglu(c, s, *_mx(32, 64), *_mx(64, 64), *_mx(3, 32))
    with pytest.raises(ValueError, match="the result"):
        ops.gemm_mx8_swiglu(c, s, *_mx(32, 64), *_mx(32, 64), *_mx(3, 64))
