"""Rows whose largest magnitude is at the ends of its type's numbers: codes and scales as they are defined."""
import pytest
import torch

from norm_reference import quantized
from peco_amd.projection import int8_linear, quantize_rows

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("channels", [8, 100, 2048])
def test_largest_and_smallest_rows(channels, dtype, announce):
    """One over a magnitude past 2^126 is subnormal; below 127 2^-126 a row counts as 0 (in fp16 no row is that small)."""
    announce()
    g = torch.Generator().manual_seed(channels)
    info, edge = torch.finfo(dtype), 127 * 2.0 ** -126
    most = [info.max, info.max / 2, info.max / 4, info.max / 8, info.tiny, 1.0]
    if dtype != torch.float16:
        most += [edge, edge * 2, edge / 2, edge * (1 - 2.0 ** -7), 2.0 ** -133]
    x = torch.rand(len(most), channels, generator=g) * 2 - 1
    x[:, channels // 2] = 1
    x = (x.double() * torch.tensor(most, dtype=torch.float64)[:, None]).to(dtype).to(DEV)
    rows, (codes, scales) = quantize_rows(x), quantized(x)
    assert torch.equal(rows.codes.cpu(), codes) and torch.equal(rows.scales.cpu(), scales)
    assert codes[:4].abs().amax(1).eq(127).all()
    weight = quantize_rows(torch.randn(24, channels, generator=g).to(DEV))
    for n in (1, len(most)):  # quantized by the product's own launch where the rows are short
        assert torch.equal(int8_linear(x[:n], weight, dtype=torch.float32),
                           int8_linear(quantize_rows(x[:n]), weight, dtype=torch.float32))
        assert torch.equal(int8_linear(x[:n], weight), int8_linear(quantize_rows(x[:n]), weight, dtype=dtype))
