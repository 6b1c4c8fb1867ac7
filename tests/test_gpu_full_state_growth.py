"""The full-precision scan with carries that grow past binary32 (a positive A):
what is zero stays zero and what is tiny grows as in the recurrence, whether a
row's tokens are stepped, run in chunks or are cut into segments."""
import pytest
import torch

from test_gpu_full_state import _inputs, _scan
from test_gpu_full_state_scales import _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,tokens", [(1, 200), (20, 300), (160, 200), (2, 4)])
@pytest.mark.parametrize("rate", [6.0, 15.0])
def test_growth_past_binary32(device, batch, tokens, rate):
    i = _inputs(device, batch, tokens, heads=4, seed=71)
    i["A"] = torch.full_like(i["A"], rate)
    i["x"], i["state"] = i["x"].clone(), i["state"].clone()
    i["x"][..., ::3] = 0.0                       # nothing is added to these channels
    i["state"][:, :, 0] = 0.0                    # nothing at all
    i["state"][:, :, 3] = 1e-38                  # grows, into binary32's range or past it
    y, state = _scan(i)
    ry, _, rs, sm = _reference(i)
    assert not bool(y[..., 0].any()) and not bool(state[:, :, 0].any())
    eps = (4 * tokens + 256) * 2.0 ** -24
    got, want = state.double()[:, :, 3], rs[:, :, 3]
    fits = want.abs() < 3.4e38
    assert bool((got[fits] - want[fits]).abs().le(eps * sm[:, :, 3][fits] + 1e-37).all())
    assert bool(torch.isinf(got[want.abs() > 3.5e38]).all())
    if tokens > 100:
        assert not bool(torch.isfinite(state[:, :, 1]).all())


@pytest.mark.parametrize("batch,tokens", [(1, 200), (20, 300), (160, 200)])
def test_one_head_grows(device, batch, tokens):
    """The other heads keep the recurrence's values."""
    i = _inputs(device, batch, tokens, heads=4, seed=72)
    clean = _scan(i)
    i["A"] = i["A"].clone()
    i["A"][2] = 15.0
    y, state = _scan(i)
    rest = [0, 1, 3]
    assert torch.equal(y[:, :, rest], clean[0][:, :, rest]) and torch.equal(state[:, rest], clean[1][:, rest])
