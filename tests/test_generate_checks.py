"""generate() refuses what it cannot draw with before it touches the request."""
import pytest
import torch

from mamba2_recall.generate import generate


class _Controller:
    """A controller that must not be reached."""
    def backbone(self, ids, reset=False):
        raise AssertionError("the request was reset")


@pytest.mark.parametrize("kw", [
    dict(temperature=-1.0), dict(top_k=-1), dict(top_k=1.5), dict(top_p=1.5), dict(min_p=-0.1), dict(temperature=True),
    dict(temperature=torch.ones(2)), dict(temperature=torch.ones(3, dtype=torch.float64)),
    dict(top_k=torch.ones(3)), dict(top_p=torch.ones(4)), dict(min_p=torch.ones(3, device="meta"))])
def test_filters(kw):
    with pytest.raises(ValueError):
        generate(_Controller(), None, torch.zeros(3, 4, dtype=torch.long), torch.zeros(3, 2), **kw)


@pytest.mark.parametrize("uniforms", [torch.zeros(3), torch.zeros(3, 0), torch.zeros(2, 2), torch.zeros(3, 2).double(),
                                      None])
def test_uniforms(uniforms):
    with pytest.raises(ValueError):
        generate(_Controller(), None, torch.zeros(3, 4, dtype=torch.long), uniforms)
