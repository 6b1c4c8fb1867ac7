"""The full-precision scan where the magnitudes inside one call lie far apart,
against the recurrence in 64 bits.

Tolerance (derived): as in test_gpu_full_state, (4 T + 256) 2^-24 of the sum of
the terms' magnitudes, and half a unit of binary16 for a readout.  It is held
by every channel, coordinate and token for itself."""
import math

import pytest
import torch

from test_gpu_full_state import _inputs, _scan

pytestmark = pytest.mark.gpu

# one row in four segments, rows in segments of two chunks, rows in one segment; the stepped call
CALLS = [(1, 200), (30, 500), (160, 130), (3, 4)]


def _reference(i):
    """(y, its magnitude, the pool after, its magnitude) in float64, all rows at once."""
    x, per = i["x"].double(), i["x"].shape[2] // i["B"].shape[2]
    v = i["dt"].double() + i["dt_bias"].double()
    dt = torch.logaddexp(v, torch.zeros_like(v))
    decay = torch.exp(dt * i["A"].double())
    s, m = i["state"].double(), i["state"].double().abs()
    ys, yms = [], []
    for t in range(x.shape[1]):
        b, c = (i[k][:, t].double().repeat_interleave(per, 1)[:, :, None] for k in "BC")
        add = (dt[:, t, :, None] * x[:, t])[..., None] * b
        s, m = s * decay[:, t, :, None, None] + add, m * decay[:, t, :, None, None] + add.abs()
        skip = i["D"].double()[:, None] * x[:, t]
        ys.append((s * c).sum(-1) + skip)
        yms.append((m * c.abs()).sum(-1) + skip.abs())
    return torch.stack(ys, 1), torch.stack(yms, 1), s, m


def _check(i, got, ref, but=None):
    """`but`: a channel whose readouts are past binary16."""
    (y, state), (ry, ym, rs, sm) = got, ref
    eps = (4 * i["x"].shape[1] + 256) * 2.0 ** -24
    bad = ~((state.double() - rs).abs() <= eps * sm + 1e-37)
    assert not bool(bad.any()), f"{int(bad.sum())} carried values off, channels {bad.nonzero()[:, 2].unique().tolist()[:8]}"
    beyond = ry.abs() >= 65520 * (1 - 2.0 ** -10)      # binary16's infinity or its largest value
    bad = ~((y.double() - ry).abs() <= ry.abs() * 2.0 ** -11 + 2.0 ** -25 + eps * ym)
    bad &= ~(beyond & ((y.double() * ry.sign() >= 65504 * (1 - 2.0 ** -9))))
    if but is not None:
        bad[..., but] = False
    assert not bool(bad.any()), f"{int(bad.sum())} readouts off, channels {bad.nonzero()[:, 3].unique().tolist()[:8]}"


@pytest.mark.parametrize("batch,tokens", CALLS)
@pytest.mark.parametrize("dt_shift", [0.0, -4.0])
def test_large_and_small_channels_side_by_side(device, batch, tokens, dt_shift):
    i = _inputs(device, batch, tokens, heads=4, seed=61, dt_shift=dt_shift)
    i["x"], i["state"] = i["x"].clone(), i["state"].clone()
    for p, scale in ((0, 1e4), (1, 1e-4)):
        i["x"][..., p::2] = (i["x"][..., p::2].float() * scale).half()
        i["state"][:, :, p::2] *= scale
    _check(i, _scan(i), _reference(i))


@pytest.mark.parametrize("batch,tokens", CALLS)
@pytest.mark.parametrize("value", [1e12, 1e30, -3e38])
def test_one_huge_carry(device, batch, tokens, value):
    """One channel's carry far above the others'; zeros stay zeros."""
    i = _inputs(device, batch, tokens, heads=4, seed=62, dt_shift=-4.0)
    i["x"], i["state"] = i["x"].clone(), i["state"].clone()
    i["A"] = i["A"] / 64
    i["state"][:, :, 7] = value
    i["state"][:, :, 9], i["x"][..., 9] = 0.0, 0.0
    got = _scan(i)
    _check(i, got, _reference(i), but=7)
    assert not bool(got[0][..., 9].any()) and not bool(got[1][:, :, 9].any())


@pytest.mark.parametrize("batch,tokens", CALLS)
@pytest.mark.parametrize("large,small", [(1e4, 1e-4), (1.5e4, 1e-6)])
def test_large_inputs_that_are_forgotten(device, batch, tokens, large, small):
    """Tokens of large inputs, then of small ones, with a decay that makes the
    early ones count for nothing at last."""
    i = _inputs(device, batch, tokens, heads=4, seed=63, dt_shift=2.0)
    x = torch.cat((i["x"][:, :40].float() * large, i["x"][:, 40:].float() * small), 1)
    i["x"] = x.clamp(-65504.0, 65504.0).half()
    i["C"] = (i["C"].float() / 64).half()
    _check(i, _scan(i), _reference(i))


@pytest.mark.parametrize("batch,tokens", CALLS)
def test_one_token_of_large_scores(device, batch, tokens):
    """A token whose B and C are large changes nothing in how exactly the others
    are read."""
    i = _inputs(device, batch, tokens, heads=4, seed=64)
    at = min(50, tokens - 1)
    for k in "BC":
        i[k] = (i[k].float() * 2.0 ** -6).half()
        i[k][:, at] = (i[k][:, at].float() * 2.0 ** 13).half()
    i["D"] = i["D"] * 0
    i["state"] = i["state"] * 0
    i["x"] = i["x"].clone()
    i["x"][:, at] = 0.0
    _check(i, _scan(i), _reference(i))
