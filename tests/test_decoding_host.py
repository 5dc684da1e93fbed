"""The decoder's checks and plans on the host."""

import pytest
import torch

from dsl_splat_amd import decoding


def test_eight_bits_off_the_device_are_refused():
    """Codes and scales that were moved to the host are not addresses for a kernel."""
    kept = decoding.QuantizedActivations(torch.zeros((4, 40), dtype=torch.int8), torch.zeros((4, 2), dtype=torch.uint8),
                                         torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        kept.dequantize()
