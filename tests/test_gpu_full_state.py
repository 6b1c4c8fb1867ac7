"""The full-precision scan against the recurrence in 64 bits, token by token.

Tolerance (derived): a carry or readout is a sum of at most T + 1 decayed
terms.  With M the same sum of the terms' magnitudes, each token's decay and
input add a few binary32 roundings (4 taken, 2^-24 each) and a sum of up to
256 products at most 256 more, so the error is at most (4 T + 256) 2^-24 M,
plus for a readout half a unit of binary16 (2^-11 relative, 2^-25 at least).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(device, batch, tokens, heads=8, dim=64, groups=2, pool=None, seed=0, f32=False, scale=1.0, dt_shift=0.0):
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)
    p = torch.float32 if f32 else torch.float16
    return dict(x=(normal(batch, tokens, heads, dim) * scale).half(), dt=normal(batch, tokens, heads).half(),
                A=-torch.exp(torch.rand(heads, generator=gen, device=device) * math.log(16.0)),
                B=normal(batch, tokens, groups, 128).half(), C=normal(batch, tokens, groups, 128).half(),
                D=normal(heads).to(p), dt_bias=(normal(heads) * 0.5 - 2.0 + dt_shift).to(p),
                state=normal(pool or batch, heads, dim, 128) * 0.5 * scale)


def _reference(i, lengths=None, slots=None):
    """(y, its magnitude, the pool after, its magnitude) in float64."""
    x = i["x"].double()
    batch, tokens, heads, dim = x.shape
    per = heads // i["B"].shape[2]
    v = i["dt"].double() + i["dt_bias"].double()
    dt = torch.logaddexp(v, torch.zeros_like(v))
    decay = torch.exp(dt * i["A"].double())
    pool, mags = i["state"].double(), i["state"].double().abs()
    y, ym = torch.zeros_like(x), torch.zeros_like(x)
    for b in range(batch):
        slot = b if slots is None else slots[b]
        if not 0 <= slot < pool.shape[0]:
            continue
        n = tokens if lengths is None else max(0, min(tokens, lengths[b]))
        s, m = pool[slot], mags[slot]
        for t in range(n):
            bt, ct = (i[k][b, t].double().repeat_interleave(per, 0)[:, None, :] for k in "BC")
            xt = x[b, t]
            a = decay[b, t][:, None, None]
            add = (dt[b, t][:, None] * xt)[..., None] * bt
            s, m = s * a + add, m * a + add.abs()
            y[b, t] = (s * ct).sum(-1) + i["D"].double()[:, None] * xt
            ym[b, t] = (m * ct.abs()).sum(-1) + (i["D"].double()[:, None] * xt).abs()
        pool[slot], mags[slot] = s, m
    return y, ym, pool, mags


def _scan(i, **kw):
    from mamba2_recall import full_state
    state = i["state"].clone()
    y, stats = full_state.scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["dt_bias"], state, **kw)
    assert stats is None
    return y, state


def _check(i, y, state, ref, tokens):
    ry, ym, rs, sm = ref
    eps = (4 * tokens + 256) * 2.0 ** -24
    bad = (y.double() - ry).abs() > ry.abs() * 2.0 ** -11 + 2.0 ** -25 + eps * ym
    assert not bool(bad.any()), f"{int(bad.sum())} readouts off"
    bad = (state.double() - rs).abs() > eps * sm + 1e-37
    assert not bool(bad.any()), f"{int(bad.sum())} carried values off"


@pytest.mark.parametrize("tokens", [1, 2, 3, 15, 16, 17, 63, 64, 65, 127, 129, 200, 300])
def test_lengths(device, tokens):
    i = _inputs(device, 2, tokens, seed=tokens)
    _check(i, *_scan(i), _reference(i), tokens)


@pytest.mark.parametrize("heads,dim,groups", [(1, 1, 1), (3, 5, 3), (4, 40, 1), (6, 33, 2), (5, 64, 5), (12, 128, 4),
                                              (2, 200, 1), (16, 64, 1), (9, 96, 3), (7, 72, 1)])
@pytest.mark.parametrize("tokens", [1, 70])
def test_head_layouts(device, heads, dim, groups, tokens):
    i = _inputs(device, 2, tokens, heads, dim, groups, seed=heads * dim, f32=True)
    _check(i, *_scan(i), _reference(i), tokens)


@pytest.mark.parametrize("tokens", [1, 9, 150])
def test_ragged_idle_and_pool(device, tokens):
    """Lengths from none to all (and outside), idle rows, carries out of order:
    nothing else in the pool changes."""
    i = _inputs(device, 6, tokens, pool=11, seed=5)
    lengths = [tokens, 0, tokens // 2, 1, tokens + 7, -3]
    slots = [7, 2, 10, -1, 0, 4]
    y, state = _scan(i, lengths=torch.tensor(lengths, dtype=torch.int32, device=device),
                     slots=torch.tensor(slots, dtype=torch.int32, device=device))
    _check(i, y, state, _reference(i, lengths, slots), tokens)
    for row, n in enumerate(lengths):
        n = max(0, min(tokens, n)) if slots[row] >= 0 else 0
        assert not bool(y[row, n:].any()), "readouts past the length must be zero"
    untouched = [s for s in range(11) if s not in (7, 10, 0)]
    assert torch.equal(state[untouched], i["state"][untouched])
    beyond = torch.tensor([11, -5, 2 ** 31 - 1, 3, -1, 1], dtype=torch.int32, device=device)
    y, state = _scan(i, slots=beyond)
    assert not bool(y[[0, 1, 2, 4]].any())
    kept = [s for s in range(11) if s not in (3, 1)]
    assert torch.equal(state[kept], i["state"][kept])


def test_strided_views(device):
    """Inputs as columns of wider projections, tokens of a longer buffer."""
    i = _inputs(device, 3, 90, seed=8)
    want = _scan(i)
    wide = dict(i)
    for k in ("x", "B", "C", "dt"):
        t = i[k]
        rows = t.flatten(2)
        buf = torch.full((3, 100, rows.shape[2] + 24), float("nan"), dtype=torch.float16, device=device)
        buf[:, 5:95, 3:3 + rows.shape[2]] = rows
        wide[k] = buf[:, 5:95, 3:3 + rows.shape[2]].unflatten(2, t.shape[2:]) if t.ndim == 4 else \
            buf[:, 5:95, 3:3 + rows.shape[2]]
    got = _scan(wide)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = dict(i, x=i["x"].transpose(2, 3).contiguous().transpose(2, 3))
    got = _scan(turned)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("cut", [1, 64, 77])
def test_one_call_or_two(device, cut):
    from mamba2_recall import full_state
    i = _inputs(device, 2, 140, seed=3)
    state = i["state"].clone()
    parts = []
    for r in (slice(0, cut), slice(cut, 140)):
        parts.append(full_state.scan(i["x"][:, r], i["dt"][:, r], i["A"], i["B"][:, r], i["C"][:, r], i["D"],
                                     i["dt_bias"], state)[0])
    _check(i, torch.cat(parts, 1), state, _reference(i), 140)


@pytest.mark.parametrize("scale,dt_shift", [(1e-4, 0.0), (300.0, 0.0), (1.0, 9.0), (1.0, -9.0), (2000.0, -4.0)])
def test_magnitudes(device, scale, dt_shift):
    """Small and large inputs, steps that forget at once or hardly at all; the
    readouts stay within binary16, the carries need not."""
    i = _inputs(device, 1, 130, seed=11, scale=scale, dt_shift=dt_shift)
    if scale > 1:
        i["C"] = (i["C"].float() / scale).half()
        i["D"] = (i["D"].float() / scale).half()
    _check(i, *_scan(i), _reference(i), 130)


@pytest.mark.parametrize("rate,tokens,scale", [(0.0, 130, 1.0), (0.4, 130, 1e-2), (1.5, 70, 1e-5), (1.5, 3, 1.0)])
@pytest.mark.parametrize("batch", [1, 20])
def test_carries_that_grow(device, rate, tokens, scale, batch):
    """A of 0 and above on every other head, the carry e^20 times as large at the end."""
    i = _inputs(device, batch, tokens, heads=4, seed=44, scale=scale)
    i["A"][::2] = rate
    y, state = _scan(i)
    ry, ym, rs, sm = _reference(i)
    beyond = ry.abs() >= 65520 * (1 + 2.0 ** -10)      # binary16's infinity, whatever the last bits
    assert torch.equal(y[beyond].double(), ry[beyond].sign() * math.inf)
    near = (ry.abs() > 65504 * (1 - 2.0 ** -10)) & ~beyond
    y = torch.where(beyond | near, ry, y.double())
    _check(i, y, state, (ry, ym, rs, sm), tokens)


@pytest.mark.parametrize("batch", [17, 48, 64])
def test_rows_out_of_order(device, batch):
    """More workgroups than compute units with ragged, equal, absent and
    impossible lengths and idle rows, in whatever order they are taken."""
    tokens = 100
    i = _inputs(device, batch, tokens, heads=64 if batch < 20 else 24, dim=64, groups=2, pool=batch + 3, seed=43)
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, tokens + 1, (batch,), generator=gen)
    lengths[:8] = torch.tensor([0, tokens, 64, 64, -5, tokens + 7, 1, tokens])
    slots = torch.randperm(batch + 3, generator=gen)[:batch]
    slots[3], slots[9] = -1, batch + 3
    kw = dict(lengths=lengths.to(torch.int32).to(device), slots=slots.to(torch.int32).to(device))
    _check(i, *_scan(i, **kw), _reference(i, **kw), tokens)


@pytest.mark.parametrize("batch,tokens", [(200, 8256), (1, 20000)])
def test_long_memory(device, batch, tokens):
    """Carries that hardly decay over many chunks, in one segment (many rows)
    and in several (one row); all batch rows stepped at once in 64 bits."""
    i = _inputs(device, batch, tokens, heads=1, dim=8, groups=1, seed=41, dt_shift=-3.0)
    i["A"] = torch.full((1,), -2.0 ** -9, device=device)
    y, state = _scan(i)
    v = i["dt"].double() + i["dt_bias"].double()
    dt = torch.logaddexp(v, torch.zeros_like(v))[..., 0]
    decay = torch.exp(dt * i["A"].double())
    s, m = i["state"].double()[:, 0], i["state"].double()[:, 0].abs()
    eps, worst = (4 * tokens + 256) * 2.0 ** -24, 0.0
    for t in range(tokens):
        x, b, c = i["x"][:, t, 0].double(), i["B"][:, t, 0].double(), i["C"][:, t, 0].double()
        add = (dt[:, t, None] * x)[..., None] * b[:, None]
        s, m = s * decay[:, t, None, None] + add, m * decay[:, t, None, None] + add.abs()
        if t % 509 == 0 or t >= tokens - 70:
            want = (s * c[:, None]).sum(-1) + i["D"].double() * x
            mag = (m * c[:, None].abs()).sum(-1) + (i["D"].double() * x).abs()
            over = (y[:, t, 0].double() - want).abs() - want.abs() * 2.0 ** -11 - 2.0 ** -25 - eps * mag
            assert float(over.max()) <= 0, f"token {t}"
            worst = max(worst, float(((y[:, t, 0].double() - want).norm() / want.norm())))
    # the binary16 rounding alone is 2^-12.2 in the mean square
    assert worst < 2.0 ** -11
    assert float((state[:, 0].double() - s).norm() / s.norm()) < 2.0 ** -19


@pytest.mark.parametrize("key", ["x", "B", "C", "dt"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_non_finite_inputs_stay_where_they_are(device, key, value):
    """A non-finite input of row 1, token 70 (head 3, group 0) changes no
    earlier token, no other row and no other group's heads."""
    i = _inputs(device, 2, 100, seed=21)
    clean = _scan(i)
    at = {"x": (1, 70, 3, 9), "B": (1, 70, 0, 9), "C": (1, 70, 0, 9), "dt": (1, 70, 3)}[key]
    i[key] = i[key].clone()
    i[key][at] = value
    y, state = _scan(i)
    ref = _reference(dict(i, **{key: torch.where(torch.isfinite(i[key]), i[key], torch.zeros_like(i[key]))}))
    ry, ym = ref[0], ref[1]
    eps = (4 * 100 + 256) * 2.0 ** -24

    def near(sel):
        return bool(((y.double() - ry)[sel].abs() <= ry[sel].abs() * 2.0 ** -11 + 2.0 ** -25 + eps * ym[sel]).all())
    assert near((slice(1, 2), slice(0, 70))), "an earlier token changed"
    assert torch.equal(y[0], clean[0][0]) and torch.equal(state[0], clean[1][0])
    assert near((1, slice(70, 100), slice(4, 8))), "another group's heads changed"
    if key == "x":   # the other channels of the head, too
        rest = [p for p in range(64) if p != 9]
        assert bool(((y.double() - ry)[1, :, 3][:, rest].abs()
                     <= ry[1, :, 3][:, rest].abs() * 2.0 ** -11 + 2.0 ** -25 + eps * ym[1, :, 3][:, rest]).all())
    if key == "C":
        assert bool(torch.isfinite(state).all())
        assert near((1, slice(71, 100))), "a readout weight must not reach later tokens"
    if not (key == "dt" and value == -math.inf):
        assert not bool(torch.isfinite(y[1, 70, 3]).all())


def test_masked_places_are_not_read(device):
    """NaN past a row's length and in an idle row reaches nothing."""
    i = _inputs(device, 3, 100, pool=4, seed=31)
    lengths = torch.tensor([37, 100, 64], dtype=torch.int32, device=device)
    slots = torch.tensor([3, -1, 0], dtype=torch.int32, device=device)
    want = _scan(i, lengths=lengths, slots=slots)
    for k in ("x", "B", "C", "dt"):
        i[k] = i[k].clone()
        i[k][0, 37:] = math.nan
        i[k][1] = math.nan
        i[k][2, 64:] = math.inf
    got = _scan(i, lengths=lengths, slots=slots)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_carry_past_32_bit_offsets(device):
    """A pool of more than 2^31 values: its last carry."""
    from mamba2_recall import full_state
    pool = 2 ** 31 // (128 * 64 * 128) + 2
    i = _inputs(device, 1, 3, heads=128, groups=8, seed=2)
    big = torch.empty(pool, 128, 64, 128, device=device)
    big[-1], big[0] = i["state"][0], 7.0
    slots = torch.tensor([pool - 1], dtype=torch.int32, device=device)
    y, _ = full_state.scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["dt_bias"], big, slots=slots)
    _check(i, y, big[-1:], _reference(i), 3)
    assert bool((big[0] == 7.0).all())
    del big
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens", [1, 200])
def test_same_bits_again_and_on_another_stream(device, tokens):
    i = _inputs(device, 2, tokens, heads=16, groups=1, seed=13)
    want = _scan(i)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _scan(i)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tokens", [1, 200])
def test_graph_replays_match_eager(device, tokens):
    from mamba2_recall import full_state
    i = _inputs(device, 2, tokens, seed=17)
    args = [i[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias")]
    state, eager = i["state"].clone(), i["state"].clone()
    full_state.scan(*args, state)
    state.copy_(i["state"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = full_state.scan(*args, state)
    state.copy_(i["state"])
    for _ in range(3):
        graph.replay()
        want, _ = full_state.scan(*args, eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(state, eager)


def test_refusals(device):
    from mamba2_recall import full_state
    i = _inputs(device, 2, 4)
    good = [i[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "state")]
    int32 = dict(dtype=torch.int32, device=device)

    def refused(index, value, **kw):
        args = list(good)
        if index is not None:
            args[index] = value
        with pytest.raises(ValueError):
            full_state.scan(*args, **kw)
    refused(0, i["x"].float())
    refused(0, i["x"][0])
    refused(0, i["x"].cpu())
    refused(0, i["x"][:, :0])
    refused(1, i["dt"][:, :3])
    refused(2, i["A"].half())
    refused(3, i["B"][..., :64])
    refused(4, i["C"].bfloat16())
    refused(5, i["D"].double())
    refused(6, i["dt_bias"][:3])
    refused(7, i["state"].half())
    refused(7, i["state"][:1])
    refused(7, i["state"].transpose(2, 3))
    refused(7, i["state"][:, :4])
    refused(None, None, slots=torch.zeros(2, dtype=torch.int64, device=device))
    refused(None, None, slots=torch.zeros(3, **int32))
    refused(None, None, lengths=torch.zeros(2, device=device))
    refused(None, None, lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        full_state.allocate_state(1, 8, 64, 64, device)
    with pytest.raises(ValueError):
        full_state.allocate_state(0, 8, 64, 128, device)
