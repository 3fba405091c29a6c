"""tlm_add_rmsnorm and tlm_mx8_quant on the GPU at the ends of what they take. Tolerances are those of test_gpu_mx8.py."""
import numpy as np
import pytest
import torch

from oracle import ref
from test_gpu_mx8 import BF16, DEV, F32, _bytes, _empty, _norm_case
from tilelang.jit.adapter.mi355x import lib, ops

pytestmark = pytest.mark.gpu

# powers of ten: mean squares that vanish in fp32, that are subnormal, about the least normal one (1.2e-38), ordinary ones, about the
# largest (3.4e38) and beyond it
POWERS = [-38, -30, -23, -22, -20, -19.5, -19, -18.9, -18, -5, 0, 12, 19, 19.2, 19.3, 20, 30, 37]


@pytest.mark.parametrize("cols", [32, 544, 2048, 4096, 8192, 16384, 32768])
@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -130])
def test_rows_whose_squares_leave_fp32(cols, stream, eps):
    """Rows of any size, next to each other, in 16 and 8 bits."""
    g = torch.Generator().manual_seed(cols)
    r = torch.randn(len(POWERS), cols, generator=g) * torch.tensor([10.0 ** p for p in POWERS])[:, None]
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(BF16)
    _norm_case(torch.zeros(r.shape, dtype=BF16), r.to(stream), w, eps, True, True)


@pytest.mark.parametrize("cols", [8192, 16384])
def test_many_rows_whose_squares_leave_fp32(cols):
    """From 512 rows on a wide row is held by fewer threads."""
    g = torch.Generator().manual_seed(cols)
    p = torch.tensor(POWERS).repeat(30)[:520]
    r = torch.randn(520, cols, generator=g) * (10.0 ** p)[:, None]
    _norm_case(r.to(BF16), None, None, 0.0, True, False)


def test_rows_without_a_mean():
    """Infinities and NaN fill their rows' blocks or rows as the formula does; zeros with eps 0 are 0 / 0."""
    x = torch.randn(4, 4096, generator=torch.Generator().manual_seed(1)).to(BF16)
    x[0, 5], x[1, 7], x[2] = float("inf"), float("nan"), 0
    y = torch.empty_like(x, device=DEV)
    codes, scales = _empty(*x.shape)
    ops.add_rmsnorm(x.to(DEV), None, None, None, 0.0, y, codes, scales)
    y = y.cpu()
    assert torch.isnan(y[0, 5]) and not y[0, :5].any() and not y[0, 6:].any()
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[3].float()).all()
    byte = ref.mx8_untile_ref(_bytes(scales), *x.shape)
    assert byte[0, 0] == 255 and (byte[0, 1:] == 1).all() and (byte[1:3] == 255).all() and (byte[3] < 255).all()
    assert np.array_equal(np.unique(_bytes(codes)[:3] & 127), [0])


@pytest.mark.parametrize("dtype", [BF16, torch.float16, F32])
def test_quant_strides(dtype):
    """Rows a multiple of 8 elements apart, 0 among them, in any 16 bytes of a buffer; what its docstring excludes is refused."""
    x = torch.randn(6, 96 + 1001, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    flat = x.flatten()
    for stride, at in ((0, 0), (8, 8), (96, 16), (104, 8), (1000, 24)):
        rows = flat.as_strided((5, 96), (stride, 1), at)
        codes, scales = ops.mx8_quant(rows, *_empty(5, 96))
        want, byte = ref.mx8_quantise_ref(rows.cpu())
        assert np.array_equal(_bytes(codes), want)
        assert np.array_equal(ref.mx8_untile_ref(_bytes(scales), 5, 96), byte)
    for stride, at in ((97, 0), (100, 0), (96, 1)):
        with pytest.raises(lib.TLMError, match="multiple of 8"):
            ops.mx8_quant(flat.as_strided((5, 96), (stride, 1), at), *_empty(5, 96))
    # a single row has no stride
    ops.mx8_quant(flat.as_strided((1, 96), (97, 1), 0), *_empty(1, 96))
