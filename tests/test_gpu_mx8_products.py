"""Products of 8-bit operands on the GPU where a variant begins or ends: every tile on operands of any value, sums that the
matrix core cuts, blocks without a number, splits side by side. Tolerances are those of test_gpu_mx8.py."""
import numpy as np
import pytest
import torch

from test_mx8_oracle import plan
from test_gpu_mx8 import ARITH, DEV, E4M3, E8M0, _check_mx, _check_unused, _device_values, _empty
from tilelang.jit.adapter.mi355x import ops

pytestmark = pytest.mark.gpu


def _rows(rows, K, g, scale=1.0):
    """Random rows, quantised."""
    x = scale * torch.randn(rows, K, generator=g, device=DEV) * torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEV))
    return ops.mx8_quant(x, *_empty(rows, K))


def _gated(a, gate, up):
    """up * silu(gate) in float64, and how far it moves when every product's magnitude is off by one part."""
    x, v, u = (_device_values(m) for m in (a, gate, up))
    v, u = v.T.contiguous(), u.T.contiguous()
    g, h = x @ v, x @ u
    gs, hs = x.abs() @ v.abs(), x.abs() @ u.abs()
    silu = g * torch.sigmoid(g)
    return (h * silu).cpu().numpy(), (silu.abs() * hs + 1.1 * h.abs() * gs).cpu().numpy()  # |silu'| < 1.1


FP32 = 2.0 ** -16  # of the products' magnitudes: K / 32 + 40 roundings of 2^-24


@pytest.mark.parametrize("M,N,K", [(1, 33024, 512), (16, 33024, 288), (32, 40960, 256)])
def test_few_rows_of_many_columns(M, N, K):
    """Up to 32 rows are summed in fp32 whatever the columns."""
    g = torch.Generator(device=DEV).manual_seed(N + M)
    a, gate, up = _rows(M, K, g), _rows(N, K, g, K ** -0.5), _rows(N, K, g, K ** -0.5)
    codes, scales = _empty(M, N)
    ops.gemm_mx8_swiglu(*a, *gate, *up, codes, scales)
    want, move = _gated(a, gate, up)
    _check_mx(codes, scales, want, FP32 * move + ARITH * np.abs(want) + 2.0 ** -126)
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
    ops.gemm_mx8_swiglu(*a, *w, *w, codes, scales)
    c = codes.view(torch.uint8)
    assert torch.equal(c, c[:1].expand_as(c))
    s = scales.view(torch.uint8).permute(0, 3, 1, 2).flatten(2).flatten(0, 1)[:M]
    assert torch.equal(s, s[:1].expand_as(s))
