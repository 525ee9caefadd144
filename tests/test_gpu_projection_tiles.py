"""Every tile of the 8-bit product over several blocks of channels, with rows, channels and outputs that end inside it."""
import pytest
import torch

from norm_reference import product
from peco_amd.projection import QuantizedRows, int8_linear

DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# rows, channels, outputs, by the tile that they take at 256 CUs
SIZES = [
    # 256 x 256 over blocks of 128 channels: 3, 5 and 9 of them, whole ones and a remainder; one round of tiles and 2.6
    (4096, 384, 4096), (4001, 640, 4001), (4090, 1111, 4088), (3999, 130, 3846), (7006, 1111, 6001),
    # 128 x 128, blocks of 128: 9, 5, 10 and 3
    (2000, 1111, 1999), (2048, 640, 2000), (1500, 1280, 2047), (1999, 384, 1998),
    # 64 x 64 with the channels over 4 wavefronts, blocks of 256: 5, 5 and 4
    (300, 1111, 1000), (1025, 1280, 1030), (200, 1000, 131),
    # few rows, segments of 256 that 8 wavefronts take in turn: 20 and 17
    (32, 5120, 100), (9, 4111, 70),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,channels,outputs", SIZES)
def test_tiles(rows, channels, outputs, dtype, announce):
    """Against the definition, and to the bit against 16 rows at a time, which another kernel takes (results do not depend on
    the other rows)."""
    announce()
    g = torch.Generator(device=DEV).manual_seed(rows + channels + outputs)
    a, w = (torch.randint(-128, 128, (n, channels), generator=g, device=DEV).to(torch.int8) for n in (rows, outputs))
    sa, sw = (torch.rand(n, generator=g, device=DEV).add_(0.1).div_(50) for n in (rows, outputs))
    bias = torch.randn(outputs, generator=g, device=DEV)
    pitch = -(-channels // 16) * 16
    wide = torch.full((outputs, pitch), 77, dtype=torch.int8, device=DEV)  # (what is behind the channels counts for nothing)
    wide[:, :channels] = w
    weight = QuantizedRows(wide[:, :channels], sw)
    wide = torch.full((rows, pitch), -99, dtype=torch.int8, device=DEV)
    wide[:, :channels] = a
    codes = wide[:, :channels]
    out = int8_linear(QuantizedRows(codes, sa), weight, bias, dtype=dtype)
    ref, bound = product(a, sa, w, sw, bias, dtype)
    assert ((out.double() - ref).abs() <= bound).all()
    if rows > 32:
        parts = [int8_linear(QuantizedRows(c, s), weight, bias, dtype=dtype) for c, s in zip(codes.split(16), sa.split(16))]
        assert torch.equal(out, torch.cat(parts))
