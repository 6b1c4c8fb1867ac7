"""Rows of different lengths through modules that the ragged convolution does
not stand for are refused before the request is touched."""
from types import SimpleNamespace

import pytest
import torch
from torch import nn

from mamba2_recall import full_state


class _OnHost(full_state.FullState):
    device, _installed = torch.device("cpu"), True

    def reset(self, batch_size=1):
        raise AssertionError("the request was reset")


class _Conv(nn.Conv1d):
    pass


def _controller(mixers):
    c = _OnHost.__new__(_OnHost)
    c._running, c._adapters, c._mixers = False, None, mixers
    c._request = SimpleNamespace(next_layer=0, failed=False)
    c.calls = []
    c.model = SimpleNamespace(backbone=lambda ids: c.calls.append(ids) or ids)
    return c


def _mixers(conv=None, act=None):
    plain = SimpleNamespace(conv1d=nn.Conv1d(8, 8, 4, groups=8, padding=3), act=nn.SiLU())
    return [plain, SimpleNamespace(conv1d=conv or plain.conv1d, act=act or plain.act)]


def _hooked(module):
    module.register_forward_hook(lambda *a: None)
    return module


@pytest.mark.parametrize("reset", [False, True])
@pytest.mark.parametrize("mixers", [
    _mixers(act=nn.GELU()), _mixers(act=_hooked(nn.SiLU())), _mixers(conv=_Conv(8, 8, 4, groups=8, padding=3)),
    _mixers(conv=_hooked(nn.Conv1d(8, 8, 4, groups=8, padding=3)))])
def test_refused_before_the_request_is_touched(mixers, reset):
    c = _controller(mixers)
    ids, lengths = torch.zeros(2, 5, dtype=torch.long), torch.tensor([5, 2], dtype=torch.int32)
    with pytest.raises(ValueError, match="plain nn.Conv1d and nn.SiLU"):
        c.backbone(ids, reset=reset, lengths=lengths)
    assert not c.calls and not c._request.failed and not c._running
    c.backbone(ids)               # rows of one length run the modules
    assert len(c.calls) == 1


def test_plain_modules_pass():
    c = _controller(_mixers())
    c.backbone(torch.zeros(2, 5, dtype=torch.long), lengths=torch.tensor([5, 2], dtype=torch.int32))
    assert len(c.calls) == 1
