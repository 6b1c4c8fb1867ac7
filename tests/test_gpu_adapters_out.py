"""`out` of the adapters' call: base itself, memory of its own, or refused."""
import pytest
import torch

from test_gpu_adapters import _add, _case

pytestmark = pytest.mark.gpu


def test_out_overlapping_base(device):
    c = _case(device, 40, 128, 64, 3, 8, seed=91)
    want = _add(c)
    buf = torch.empty(41, 64, dtype=torch.float16, device=device)
    base = buf[:40].copy_(c["base"])
    for out in (buf[1:], buf.view(-1)[3:3 + 40 * 64].view(40, 64)):   # rows that others still read
        with pytest.raises(ValueError):
            _add(dict(c, base=base), out=out)
    wide = torch.empty(40, 100, dtype=torch.float16, device=device)
    wide[:, :64] = c["base"]
    with pytest.raises(ValueError):   # dense rows in the memory of wider ones
        _add(dict(c, base=wide[:, :64]), out=wide.view(-1)[:40 * 64].view(40, 64))
    assert torch.equal(base, c["base"])
    assert torch.equal(_add(dict(c, base=base), out=base), want)
    own = torch.empty_like(c["base"])
    assert _add(c, out=own) is own and torch.equal(own, want)


def test_out_in_the_memory_of_x(device):
    """x has been read when the first output is written."""
    c = _case(device, 40, 64, 64, 3, 8, seed=92)
    want = _add(c)
    x = c["x"].clone()
    assert torch.equal(_add(dict(c, x=x), out=x), want)


def test_out_between_the_rows_of_base(device):
    """Memory inside a wider buffer that no row of base covers."""
    c = _case(device, 3, 96, 32, 2, 8, seed=93)
    want = _add(c)
    wide = torch.empty(3, 200, dtype=torch.float16, device=device)
    wide[:, :32] = c["base"]
    out = wide.view(-1)[200 + 40:200 + 40 + 96].view(3, 32)
    assert torch.equal(_add(dict(c, base=wide[:, :32]), out=out), want)
    for start in (200 + 31, 400 - 95, 169 - 64):   # one element of a row
        with pytest.raises(ValueError):
            _add(dict(c, base=wide[:, :32]), out=wide.view(-1)[start:start + 96].view(3, 32))
