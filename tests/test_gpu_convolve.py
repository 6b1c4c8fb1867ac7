"""The ragged convolution over a pool of windows (full_state.convolve) against
the formula in binary64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

MODEL = (8192, 1024, 1024)


def _inputs(device, batch, tokens, sizes, pool, seed=0, pad=0, scale=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    c = sum(sizes)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)
    value = (normal(batch, tokens, c + pad) * scale).half()[..., :c]
    window = normal(pool, 4, c).half().permute(0, 2, 1)
    return value, (normal(c, 4) * 0.4).half(), (normal(c) * 0.1).half(), window


def _oracle(value, weight, bias, window, lengths, slots, silu=True):
    """(outputs, sum of the terms' magnitudes, windows) in binary64 on the host, row by row."""
    value, weight, window = value.double().cpu(), weight.double().cpu(), window.double().cpu().clone()
    batch, tokens, c = value.shape
    out, size = torch.zeros(batch, tokens, c, dtype=torch.float64), torch.zeros(batch, tokens, c, dtype=torch.float64)
    b64 = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double().cpu()
    for i in range(batch):
        slot = i if slots is None else int(slots[i])
        n = tokens if lengths is None else max(0, min(tokens, int(lengths[i])))
        if not 0 <= slot < window.shape[0] or n == 0:
            continue
        series = torch.cat((window[slot].T, value[i, :n]), 0)                  # [4 + n, C]
        terms = torch.stack([series[1 + j:1 + j + n] * weight[:, j] for j in range(4)])
        s = terms.sum(0) + b64
        out[i, :n] = s * torch.sigmoid(s) if silu else s
        size[i, :n] = terms.abs().sum(0) + b64.abs()
        window[slot] = series[-4:].T
    return out, size, window


def _check(device, value, weight, bias, window, sizes, lengths=None, slots=None, silu=True):
    from mamba2_recall import full_state
    want, size, windows = _oracle(value, weight, bias, window, lengths, slots, silu)
    parts = full_state.convolve(value, weight, bias, window, sizes, lengths=lengths, slots=slots, silu=silu)
    assert [tuple(p.shape) for p in parts] == [(*value.shape[:2], n) for n in sizes]
    assert all(p.is_contiguous() for p in parts)
    got = torch.cat(parts, -1).double().cpu()
    # half a step of binary16 (2^-25 among its subnormals); five binary32 roundings of sums no
    # larger than the terms' magnitudes, through a SiLU of slope up to 1.1; 2^-19 for its exponential
    bound = want.abs() * (2.0 ** -11 + 2.0 ** -19) + 2.0 ** -25 + 5 * 1.1 * 2.0 ** -24 * size
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), (got - want).abs().max())
    assert torch.equal(window.double().cpu(), windows)
    return parts


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 77, 500])
@pytest.mark.parametrize("batch", [1, 3])
def test_lengths(device, batch, tokens):
    _check(device, *_inputs(device, batch, tokens, MODEL, batch, pad=8320), MODEL)


@pytest.mark.parametrize("sizes", [(1, 1, 1), (3, 5, 7), (8, 8, 8), (40, 16, 8), (960, 384, 384), (2049, 130, 64),
                                   (4096, 512, 512), (16384, 1024, 1024)])
@pytest.mark.parametrize("tokens", [1, 6, 33])
def test_channels(device, sizes, tokens):
    _check(device, *_inputs(device, 2, tokens, sizes, 3, seed=1), sizes, slots=torch.tensor([2, 0], dtype=torch.int32,
                                                                                           device=device))


@pytest.mark.parametrize("sizes", [(64, 16, 16), (33, 6, 9)])
@pytest.mark.parametrize("tokens", [1, 3, 21])
def test_ragged_rows_and_idle_rows(device, sizes, tokens):
    counts = [tokens, 0, 1, 2, tokens - 1, 5, -3, tokens + 9, 4, 3]
    lengths = torch.tensor(counts, dtype=torch.int32, device=device)
    slots = torch.tensor([4, 9, -1, 2, 0, 11, 5, 7, 50, 3], dtype=torch.int32, device=device)
    value, weight, bias, window = _inputs(device, 10, tokens, sizes, 12, seed=2)
    before = window.clone()
    parts = _check(device, value, weight, bias, window, sizes, lengths, slots)
    # rows that nothing names, idle rows and empty rows keep their windows
    for slot in (1, 5, 6, 8, 9, 10):
        assert torch.equal(window[slot], before[slot])
    for i, n in enumerate(counts):
        for p in parts:
            assert not bool(p[i, max(0, min(tokens, n)):].any())


def test_strides_and_alignment(device):
    sizes = (64, 16, 16)
    value, weight, bias, window = _inputs(device, 3, 11, sizes, 3, seed=3)
    apart = torch.empty(11, 3, 97, dtype=torch.float16, device=device)   # rows of an odd stride, tokens before rows
    view = apart[..., 1:].transpose(0, 1)
    view.copy_(value)
    store = torch.zeros(3, 5, 99, dtype=torch.float16, device=device)
    odd = store[:, 1:, 2:98].permute(0, 2, 1)
    odd.copy_(window)
    first = _check(device, value, weight, bias, window, sizes)
    second = _check(device, view, weight, bias, odd, sizes)
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    assert not bool(store[:, 0].any()) and not bool(store[:, :, :2].any()) and not bool(store[:, :, 98].any())
    # a value whose channels are apart, a weight that is a view, no bias, no SiLU
    wide = torch.empty(3, 11, 96, 2, dtype=torch.float16, device=device)[..., 0]
    wide.copy_(value)
    taps = torch.empty(96, 1, 5, dtype=torch.float16, device=device)[:, 0, 1:]
    taps.copy_(weight)
    _check(device, wide, taps, None, window, sizes, silu=False)


def test_pieces_equal_one_call(device):
    """A row's outputs and window do not depend on how its tokens are split."""
    from mamba2_recall import full_state
    sizes = (96, 32, 32)
    value, weight, bias, window = _inputs(device, 2, 40, sizes, 2, seed=4)
    pieces = window.clone(memory_format=torch.preserve_format)
    whole = full_state.convolve(value, weight, bias, window, sizes)
    for lo, hi in ((0, 1), (1, 2), (2, 5), (5, 21), (21, 24), (24, 40)):
        part = full_state.convolve(value[:, lo:hi], weight, bias, pieces, sizes)
        assert all(torch.equal(p, w[:, lo:hi]) for p, w in zip(part, whole))
    assert torch.equal(pieces, window)


def test_extreme_values(device):
    """Large sums saturate as the formula does; a non-finite input reaches its
    own and the next three tokens of its channel and nothing else."""
    from mamba2_recall import full_state
    sizes = (16, 8, 8)
    value, weight, bias, window = _inputs(device, 1, 24, sizes, 1, seed=5, scale=60.0)
    _check(device, value, weight, bias, window, sizes)
    clean = full_state.convolve(value, weight, bias, full_state.allocate_windows(1, 32, device), sizes)
    for bad in (float("nan"), float("inf"), float("-inf")):
        broken = value.clone()
        broken[0, 9, 5] = bad
        got = full_state.convolve(broken, weight, bias, full_state.allocate_windows(1, 32, device), sizes)
        want = clean[0].clone()
        touched = torch.zeros_like(want, dtype=torch.bool)
        touched[0, 9:13, 5] = True
        assert torch.equal(got[0][~touched], want[~touched])
        assert torch.equal(got[1], clean[1]) and torch.equal(got[2], clean[2])
        if bad != bad:
            assert bool(torch.isnan(got[0][touched]).all())
        assert not bool((got[0][touched] == want[touched]).any())


def test_other_stream_and_graph(device):
    from mamba2_recall import full_state
    sizes = (128, 32, 32)
    value, weight, bias, window = _inputs(device, 4, 19, sizes, 6, seed=6)
    slots = torch.tensor([5, -1, 0, 2], dtype=torch.int32, device=device)
    lengths = torch.tensor([19, 4, 1, 7], dtype=torch.int32, device=device)
    first = window.clone(memory_format=torch.preserve_format)
    want = full_state.convolve(value, weight, bias, window, sizes, lengths=lengths, slots=slots)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    static = first.clone(memory_format=torch.preserve_format)
    with torch.cuda.stream(stream):
        side = full_state.convolve(value, weight, bias, static, sizes, lengths=lengths, slots=slots)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, want)) and torch.equal(static, window)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = full_state.convolve(value, weight, bias, static, sizes, lengths=lengths, slots=slots)
    for _ in range(3):
        static.copy_(first)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(static, window)


def test_long_row(device):
    """Offsets past 2^31 elements."""
    from mamba2_recall import full_state
    sizes, tokens = (8192, 1024, 1024), 230001
    gen = torch.Generator(device=device).manual_seed(7)
    value = torch.empty(1, tokens, 10240, dtype=torch.float16, device=device)
    value.normal_(generator=gen)
    weight = (torch.randn(10240, 4, generator=gen, device=device) * 0.4).half()
    window = full_state.allocate_windows(1, 10240, device)
    parts = full_state.convolve(value, weight, None, window, sizes)
    assert torch.equal(window[0].T, value[0, -4:])
    tail = full_state.allocate_windows(1, 10240, device)
    tail[0].copy_(value[0, -30:-26].T)
    last = full_state.convolve(value[:, -26:], weight, None, tail, sizes)
    assert all(torch.equal(p[:, -26:], q) for p, q in zip(parts, last))


@pytest.mark.parametrize("tokens", [97, 128, 131])
def test_many_workgroups(device, tokens):
    """Enough rows for 32 tokens a thread: whole and ragged runs, idle rows."""
    sizes, batch = (64, 16, 16), 70
    value, weight, bias, window = _inputs(device, batch, tokens, sizes, 80, seed=9, pad=32)
    gen = torch.Generator(device=device).manual_seed(10)
    slots = torch.randperm(80, generator=gen, device=device)[:batch].to(torch.int32)
    slots[::17] = -1
    lengths = torch.randint(0, tokens + 1, (batch,), generator=gen, device=device, dtype=torch.int32)
    lengths[:6] = torch.tensor([tokens, 32, 33, 31, 64, 96], dtype=torch.int32, device=device)
    _check(device, value, weight, bias, window, sizes, lengths, slots)
    _check(device, value, weight, bias, window, sizes)


@pytest.mark.parametrize("sizes", [(64, 16, 16), (33, 6, 9)])
@pytest.mark.parametrize("tokens", [1, 7, 45])
def test_what_stands_behind_a_row_does_not_count(device, sizes, tokens):
    """NaN and infinities behind the rows' lengths, in the windows of idle and empty rows and in the
    window's first place reach nothing."""
    counts = torch.tensor([tokens, tokens // 2, 1, 0, tokens], dtype=torch.int32, device=device)
    slots = torch.tensor([0, 1, 2, 3, -1], dtype=torch.int32, device=device)
    value, weight, bias, window = _inputs(device, 5, tokens, sizes, 5, seed=9)
    dirty, windows = value.clone(), window.clone()
    windows[:, :, 0] = float("nan")
    windows[3:] = float("inf")
    for i, n in enumerate((tokens, tokens // 2, 1, 0, 0)):
        dirty[i, n:] = float("nan") if i % 2 else float("-inf")
    want = _check(device, value, weight, bias, window, sizes, counts, slots)
    from mamba2_recall import full_state
    got = full_state.convolve(dirty, weight, bias, windows, sizes, lengths=counts, slots=slots)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    live = [i for i, n in enumerate(counts[:3].tolist()) if n]
    # (a window of fewer than four tokens shifts: its first place goes)
    assert torch.equal(windows[live], window[live]) and bool(torch.isinf(windows[3:]).all())
