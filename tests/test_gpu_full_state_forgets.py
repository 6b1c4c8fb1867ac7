"""The full-precision scan with decays that leave nothing (A far below 0, minus
infinity among them): each token stands alone, in every way a call is run."""
import math

import pytest
import torch

from test_gpu_full_state import _inputs, _scan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,tokens", [(1, 200), (160, 130), (2, 4)])
@pytest.mark.parametrize("rate", [-1e6, -1e30, -1e37, -3e38, -math.inf])
def test_every_token_alone(device, batch, tokens, rate):
    """y = (dt C.B + D) x; the carry is the last token's addition.  Tolerance: a
    sum of 128 products and a few roundings in binary32 (256 2^-24 of the sum of
    magnitudes), half a unit of binary16."""
    i = _inputs(device, batch, tokens, heads=4, seed=95)
    i["A"] = torch.full_like(i["A"], rate)
    y, state = _scan(i)
    v = i["dt"].double() + i["dt_bias"].double()
    dt = torch.logaddexp(v, torch.zeros_like(v))[..., None]
    b, c = (i[k].double().repeat_interleave(2, 2) for k in "BC")
    x, skip = i["x"].double(), i["D"].double()[:, None]
    weight, size = dt * (b * c).sum(-1, keepdim=True), dt * (b * c).abs().sum(-1, keepdim=True)
    want, mag = (weight + skip) * x, (size + skip.abs()) * x.abs()
    bad = ~((y.double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -25 + 256 * 2.0 ** -24 * mag)
    assert not bool(bad.any()), f"{int(bad.sum())} readouts off"
    last = (dt * x)[:, -1, :, :, None] * b[:, -1, :, None]
    bad = ~((state.double() - last).abs() <= 256 * 2.0 ** -24 * last.abs() + 1e-37)
    assert not bool(bad.any()), f"{int(bad.sum())} carried values off"
