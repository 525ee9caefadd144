"""The modules around a block's attention, as far as they go without a GPU: what they refuse, what they keep and what they
leave alone."""
import pytest
import torch

from peco_amd.norm import LayerNorm


@pytest.mark.parametrize("affine", [True, False])
def test_a_layer_norm_takes_rows_of_its_own_channels(affine):
    norm = LayerNorm(64, elementwise_affine=affine)
    for shape in ((128,), (2, 32), (64, 3), ()):
        with pytest.raises(ValueError, match="64 channels"):
            norm(torch.zeros(shape))
    with pytest.raises(ValueError, match="GPU"):  # rows of its channels come as far as the device
        norm(torch.zeros(2, 64))
