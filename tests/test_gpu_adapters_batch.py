"""Adapters for another number of requests than a call has are refused before
the request is touched."""
import pytest
import torch

from test_gpu_generate import BATCH, VOCAB, _few, _sets, small  # noqa: F401  (small: a fixture)

pytestmark = pytest.mark.gpu


def test_refused_call_leaves_the_request(small, device):  # noqa: F811
    from mamba2_recall.full_state import FullState
    gen = torch.Generator(device=device).manual_seed(4)
    prompt = torch.randint(0, VOCAB, (BATCH, 9), generator=gen, device=device)
    sets = [None, dict(out_proj=_sets(device)[1]["out_proj"])]       # the last projection of all
    with _few(FullState, small) as c:
        c.backbone(prompt[:, :8], reset=True)
        want = c.backbone(prompt[:, 8:])
        c.backbone(prompt[:, :8], reset=True)
        c.use_adapters(sets, torch.zeros(BATCH - 1, dtype=torch.int32, device=device))
        for reset in (False, True):
            with pytest.raises(ValueError, match="batch"):
                c.backbone(prompt[:, 8:], reset=reset)
        c.use_adapters(None)
        assert c.cache_breakdown()["tokens_per_layer"] == [8, 8]
        assert torch.equal(c.backbone(prompt[:, 8:]), want)
