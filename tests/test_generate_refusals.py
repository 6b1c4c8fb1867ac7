"""What generate() can refuse before it touches the request, it refuses there:
masks whose type, device, axes or rows are wrong, and a prompt that the
penalties cannot count."""
import pytest
import torch

from mamba2_recall import sampling
from mamba2_recall.generate import generate

I32 = torch.int32


class _Controller:
    """A controller that must not be reached."""
    def backbone(self, *args, **kw):
        raise AssertionError("the request was reset")


@pytest.mark.parametrize("allowed", [
    torch.zeros(2, dtype=torch.int64), torch.zeros(3, 2), torch.zeros(2, 2, dtype=I32), torch.zeros(4, 2, dtype=I32),
    torch.zeros(0, 2, dtype=I32), torch.zeros(0, dtype=I32), torch.zeros((), dtype=I32), torch.zeros(3, 2, 2, dtype=I32),
    torch.zeros(3, 0, dtype=I32), torch.zeros(3, 2, dtype=torch.bool)])
def test_masks(allowed):
    with pytest.raises(ValueError, match="allowed|mask"):
        generate(_Controller(), None, torch.zeros(3, 4, dtype=torch.long), torch.zeros(3, 2), allowed=allowed)


@pytest.mark.parametrize("kw", [dict(repetition=1.1), dict(presence=0.5), dict(frequency=torch.zeros(3))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.int16, torch.uint8])
def test_prompts_that_cannot_be_counted(dtype, kw):
    with pytest.raises(ValueError, match="prompt must be int64 or int32"):
        generate(_Controller(), None, torch.zeros(3, 4, dtype=dtype), torch.zeros(3, 2), **kw)


def test_good_settings_reach_the_request():
    prompt, uniforms = torch.zeros(3, 4, dtype=torch.long), torch.zeros(3, 2)
    for kw in (dict(allowed=torch.zeros(2, dtype=I32)), dict(allowed=torch.zeros(3, 2, dtype=I32)), dict(allowed=lambda drawn: None),
               dict(repetition=1.1, presence=torch.zeros(3)), dict(allowed=torch.zeros(3, 4, dtype=I32)[:, ::2])):
        with pytest.raises(AssertionError, match="the request was reset"):
            generate(_Controller(), None, prompt, uniforms, **kw)


def test_masks_of_an_unknown_vocabulary():
    """Every check but the one of the words' number, which the logits bring."""
    like = torch.zeros(3, 40)
    with pytest.raises(ValueError):
        sampling.masks(like, 40, torch.zeros(3, dtype=I32), None)
    one, rows = sampling.masks(like, None, torch.zeros(3, dtype=I32), None)
    assert one.shape == (3, 3) and rows is None
