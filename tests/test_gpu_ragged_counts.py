"""What a controller counts for rows of different lengths: the places that each
layer was called with, padding among them."""
import pytest

from test_gpu_generate import LAYERS, _few, small  # noqa: F401  (small: a fixture)
from test_gpu_generate_queue import _int32, _prompts

pytestmark = pytest.mark.gpu


def test_places_and_not_tokens_are_counted(small, device):  # noqa: F811
    from mamba2_recall.full_state import FullState
    prompt, _ = _prompts(device, 20, seed=13)
    with _few(FullState, small) as c:
        c.backbone(prompt, reset=True, lengths=_int32(device, 3, 20, 0))
        assert c.cache_breakdown()["tokens_per_layer"] == [20] * LAYERS
        c.backbone(prompt[:, :4], lengths=_int32(device, 0, 0, 1))
        c.backbone(prompt[:, :1])
        assert c.cache_breakdown()["tokens_per_layer"] == [25] * LAYERS
