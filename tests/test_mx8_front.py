"""The Python front of the 8-bit operands, without a GPU."""
import pytest
import torch

from tilelang.jit.adapter.mi355x import ops


def test_tile_scales_takes_bytes_only():
    """Wider scales of one block would be read as four bytes each and pass for the tiled scales of K 32."""
    for bad in (torch.ones(64, 1), torch.ones(64, 1).half(), torch.ones(64, 1, dtype=torch.int32), torch.ones(64).byte(),
                torch.ones(2, 64, 1).byte()):
        with pytest.raises(ValueError, match="bytes"):
            ops.mx8_tile_scales(bad)
    for dtype in (torch.uint8, torch.float8_e8m0fnu):
        t = ops.mx8_tile_scales(torch.full((64, 1), 127, dtype=torch.uint8).view(dtype))
        assert t.shape == ops.mx8_scales_shape(64, 32)
        assert (t.view(torch.uint8)[0, 0, 0] == 127).all()
