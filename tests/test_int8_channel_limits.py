"""The channels that a projection in 8-bit integers may have are checked when
its weights are laid out, before anything is allocated."""
import pytest
import torch

from mamba2_recall import int8


class _OnDevice(torch.Tensor):
    """A tensor of host memory (one element) that says it is on the GPU: the
    checks in front of the first allocation need no more."""
    is_cuda = True


def _wide(n, dtype):
    return torch.zeros(1, 1, dtype=dtype).expand(n, 1).as_subclass(_OnDevice)


@pytest.mark.parametrize("n", [(1 << 24) + 1, 1 << 25, 1 << 40])
def test_more_channels_than_a_product_takes(n):
    with pytest.raises(ValueError, match="16777216 channels"):
        int8.Int8Weight(_wide(n, torch.int8), torch.zeros(1).expand(n))


@pytest.mark.parametrize("n", [(1 << 24) - 127, 1 << 24, (1 << 24) + 1, 1 << 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_more_channels_than_one_launch_forms(n, dtype):
    with pytest.raises(ValueError, match="16777088 channels"):
        int8.Int8Weight.quantize(_wide(n, dtype))
