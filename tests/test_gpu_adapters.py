"""Adapters of many requests against the formula in 64 bits.

Tolerance (derived): sums of K and of rank products in binary32, each product
and sum rounded, give at most (K + rank + 8) 2^-24 of the sum of magnitudes,
and the result one binary16 rounding (2^-11 relative, 2^-25 at least)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(device, rows, k, n, count, rank, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)
    return dict(x=normal(rows, k).half(), base=normal(rows, n).half(), down=(normal(count, rank, k) / k ** 0.5).half(),
                up=(normal(count, n, rank) / rank ** 0.5).half(),
                scale=torch.rand(count, generator=gen, device=device) + 0.5,
                ids=torch.randint(-1, count, (rows,), generator=gen, device=device).to(torch.int32))


def _reference(c):
    out, mag = c["base"].double(), torch.zeros_like(c["base"], dtype=torch.float64)
    for a in range(c["down"].shape[0]):
        rows = (c["ids"] == a).nonzero()[:, 0]
        x, d, u, s = c["x"][rows].double(), c["down"][a].double(), c["up"][a].double(), c["scale"][a].double()
        out[rows] += s * ((x @ d.T) @ u.T)
        mag[rows] = s.abs() * ((x.abs() @ d.abs().T) @ u.abs().T)
    return out, mag


def _check(c, got):
    from mamba2_recall import adapters  # noqa: F401
    want, mag = _reference(c)
    eps = (c["x"].shape[1] + c["down"].shape[1] + 8) * 2.0 ** -24
    bad = (got.double() - want).abs() > want.abs() * 2.0 ** -11 + 2.0 ** -25 + eps * mag
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outputs off"


def _add(c, **kw):
    from mamba2_recall import adapters
    return adapters.add(c["base"], c["x"], adapters.AdapterSet(c["down"], c["up"], c["scale"]), c["ids"], **kw)


@pytest.mark.parametrize("rows", [1, 2, 3, 15, 16, 17, 64, 65, 130, 300])
@pytest.mark.parametrize("rank", [1, 8, 16])
def test_rows(device, rows, rank):
    c = _case(device, rows, 512, 384, 5, rank, seed=rows)
    _check(c, _add(c))


@pytest.mark.parametrize("k,n", [(1, 1), (7, 13), (64, 64), (100, 250), (2050, 515), (4096, 33), (33, 4096), (1000, 1000)])
@pytest.mark.parametrize("rank", [3, 20, 64, 256])
@pytest.mark.parametrize("rows", [5, 70])
def test_sizes(device, rows, k, n, rank):
    c = _case(device, rows, k, n, 3, rank, seed=k + n)
    _check(c, _add(c))


@pytest.mark.parametrize("rank", [9, 32, 48])
def test_many_rows(device, rank):
    """More rows than one tile at a time is for, an odd number of tiles; every
    row its own adapter, and runs of rows with one."""
    c = _case(device, 4120, 200, 136, 7, rank, seed=rank)
    _check(c, _add(c))
    c["ids"] = (torch.arange(4120, device=device) // 311 % 9 - 1).to(torch.int32)
    _check(c, _add(c))


@pytest.mark.parametrize("rows", [1, 40, 500])
def test_requests_side_by_side(device, rows):
    """Rows of a request next to each other, changes inside a tile."""
    c = _case(device, rows, 1024, 768, 6, 16, seed=4)
    c["ids"] = (torch.arange(rows, device=device) * 7 // rows - 1).to(torch.int32)
    _check(c, _add(c))
    c["ids"] = torch.full((rows,), 2, dtype=torch.int32, device=device)
    _check(c, _add(c))


@pytest.mark.parametrize("rows", [9, 200])
def test_no_adapter_is_a_copy(device, rows):
    c = _case(device, rows, 256, 320, 4, 8, seed=6)
    c["ids"][:] = -1
    c["ids"][rows // 2] = 4        # not below the count
    c["ids"][rows // 3] = -2 ** 31
    c["x"][:] = math.nan
    assert torch.equal(_add(c), c["base"])
    c["ids"][1] = 0
    got = _add(c)
    rest = [i for i in range(rows) if i != 1]
    assert torch.equal(got[rest], c["base"][rest]) and bool(got[1].isnan().all())


def test_non_finite_rows_stay_apart(device):
    """A row of NaN changes no other row of its adapter or tile."""
    c = _case(device, 48, 512, 256, 2, 16, seed=9)
    c["ids"] = (torch.arange(48, device=device) // 24).to(torch.int32)
    clean = _add(c)
    c["x"][5, 3] = math.nan
    c["x"][30, 7] = math.inf
    got = _add(c)
    rest = [i for i in range(48) if i not in (5, 30)]
    assert torch.equal(got[rest], clean[rest])
    assert bool(got[5].isnan().all()) and not bool(torch.isfinite(got[30]).all())


@pytest.mark.parametrize("rank", [1, 3, 8])
def test_infinite_hidden_values(device, rank):
    """An infinity comes out as in the formula, also where the rank is padded."""
    c = _case(device, 20, 100, 70, 2, rank, seed=10)
    c["x"][4, 9] = math.inf
    c["x"][7, 11] = -math.inf
    c["ids"][4], c["ids"][7] = 0, 1
    c["up"] = c["up"].abs() + 0.5
    c["down"] = c["down"].abs() + 0.5     # all hidden values of a row share the sign
    got, (want, _) = _add(c), _reference(c)
    assert bool((got[4] == math.inf).all()) and bool((got[7] == -math.inf).all())
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))


@pytest.mark.parametrize("rank", [8, 5])
def test_weights_off_a_16_byte_boundary(device, rank):
    c = _case(device, 20, 64, 40, 3, rank, seed=11)
    want = _add(c)
    off = dict(c)
    for key in ("down", "up"):
        buf = torch.empty(c[key].numel() + 3, dtype=torch.float16, device=device)
        off[key] = buf[3:].view(c[key].shape).copy_(c[key])
    assert torch.equal(_add(off), want)


@pytest.mark.parametrize("scale", [1e-4, 200.0])
def test_magnitudes(device, scale):
    c = _case(device, 20, 1024, 256, 3, 16, seed=12)
    c["x"] = (c["x"].float() * scale).half()
    c["scale"] = c["scale"] / scale
    _check(c, _add(c))
    c["up"], c["scale"] = (c["up"].float() / 256).half(), c["scale"] * 256
    _check(c, _add(c))


def test_hidden_values_past_binary16(device):
    """Hidden values above 65504, brought back by a small `up`."""
    c = _case(device, 20, 1024, 256, 3, 16, seed=14)
    c["x"] = (c["x"].float() * 2000).half()
    c["down"] = (c["down"].float() * 500).half()
    c["up"] = (c["up"].float() * 2.0 ** -13).half()
    c["scale"] = c["scale"] * 2.0 ** -6
    _check(c, _add(c))


def test_views_shapes_and_out(device):
    c = _case(device, 24, 512, 256, 3, 16, seed=15)
    want = _add(c)
    wide = dict(c)
    for key in ("x", "base"):
        buf = torch.full((24, c[key].shape[1] + 9), math.nan, dtype=torch.float16, device=device)
        buf[:, 5:5 + c[key].shape[1]] = c[key]
        wide[key] = buf[:, 5:5 + c[key].shape[1]]
    assert torch.equal(_add(wide), want)
    cube = dict(c, x=c["x"].reshape(2, 12, -1), base=c["base"].reshape(2, 12, -1), ids=c["ids"].reshape(2, 12))
    assert torch.equal(_add(cube), want.reshape(2, 12, -1))
    turned = dict(c, x=c["x"].t().contiguous().t())
    assert torch.equal(_add(turned), want)
    own = c["base"].clone()
    assert _add(dict(c, base=own), out=own) is own and torch.equal(own, want)
    empty = dict(c, x=c["x"][:0], base=c["base"][:0], ids=c["ids"][:0])
    assert _add(empty).shape == (0, 256)


@pytest.mark.parametrize("rows", [4, 100])
def test_stream_and_graph(device, rows):
    from mamba2_recall import adapters
    c = _case(device, rows, 1024, 512, 3, 16, seed=16)
    want = _add(c)
    handle = adapters.AdapterSet(c["down"], c["up"], c["scale"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = adapters.add(c["base"], c["x"], handle, c["ids"])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = adapters.add(c["base"], c["x"], handle, c["ids"])
    for _ in range(3):
        out.zero_()
        graph.replay()
        want = adapters.add(c["base"], c["x"], handle, c["ids"])
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(device):
    from mamba2_recall import adapters
    c = _case(device, 4, 64, 32, 2, 8)
    s = adapters.AdapterSet(c["down"], c["up"])
    assert (s.count, s.rank, s.features) == (2, 8, (64, 32)) and bool((s.scale == 1).all())
    for down, up, scale in ((c["down"].float(), c["up"], None), (c["down"][0], c["up"], None),
                            (c["down"], c["up"][:1], None), (c["down"], c["up"][..., :4], None),
                            (c["down"].cpu(), c["up"].cpu(), None), (c["down"], c["up"], c["scale"].half()),
                            (c["down"], c["up"], c["scale"][:1]), (c["down"][:0], c["up"][:0], None)):
        with pytest.raises(ValueError):
            adapters.AdapterSet(down, up, scale)
    with pytest.raises(ValueError):
        adapters.AdapterSet(c["down"].repeat(1, 40, 1), c["up"].repeat(1, 1, 40))
    bad = [(c["base"].float(), c["x"], c["ids"]), (c["base"], c["x"][:, :32], c["ids"]), (c["base"][:3], c["x"], c["ids"]),
           (c["base"], c["x"], c["ids"].long()), (c["base"], c["x"], c["ids"][:3]), (c["base"], c["x"].cpu(), c["ids"]),
           (c["base"], c["x"], c["ids"].cpu())]
    for base, x, ids in bad:
        with pytest.raises(ValueError):
            adapters.add(base, x, s, ids)
    with pytest.raises(ValueError):
        adapters.add(c["base"], c["x"], c["down"], c["ids"])
    with pytest.raises(ValueError):
        adapters.add(c["base"], c["x"], s, c["ids"], out=c["base"].float())
