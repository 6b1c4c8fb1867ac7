"""A non-finite B, C or dt of one token leaves the other tokens of its chunk as
exact as they were (the full-precision scan; the tolerance is
test_gpu_full_state's)."""
import math

import pytest
import torch

from test_gpu_full_state import _inputs, _reference, _scan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("key", ["B", "C", "dt"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("scale", [2.0 ** -14, 2.0 ** 5])
def test_non_finite_inputs_set_no_scale(device, key, value, scale):
    """Weights (dt C.B) of about 2^-25 and of about 2^13, inputs the other way
    round, in a chunk with one non-finite value at token 70."""
    i = _inputs(device, 1, 100, seed=81)
    for k in "BC":
        i[k] = (i[k].float() * scale).half()
    i["x"] = (i["x"].float() * (4096.0 if scale < 1 else 2.0 ** -7)).half()
    i["D"], i["state"] = i["D"] * 0, i["state"] * 0
    clean = _reference(i)
    at = {"B": (0, 70, 0, 9), "C": (0, 70, 0, 9), "dt": (0, 70, 3)}[key]
    i[key] = i[key].clone()
    i[key][at] = value
    y, _ = _scan(i)
    ry, ym = clean[0], clean[1]
    eps = (4 * 100 + 256) * 2.0 ** -24
    ok = (y.double() - ry).abs() <= ry.abs() * 2.0 ** -11 + 2.0 ** -25 + eps * ym
    assert bool(ok[0, :70].all()), "an earlier token changed"
    if key == "C":
        assert bool(ok[0, 71:].all()), "a later token changed"
