"""Products in 8-bit integers whose inputs are split among workgroups: the
partial sums and tickets of every row-tile count, in graphs, on streams of
their own, and against the same rows unsplit."""
import pytest
import torch

gpu = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
FAKE = 1 << 20   # an aligned address that is not read

# rows, channels, inputs, workgroups that share a block's inputs
CASES = [
    # one, two, four and eight row tiles in k_int8_few
    (1, 40, 32768, 8), (3, 96, 16400, 4), (9, 4096, 8192, 2), (16, 1000, 32768, 8), (25, 2048, 8192, 2), (30, 500, 32768, 8),
    (40, 72, 12800, 3), (50, 4096, 8192, 2), (64, 1024, 32768, 8), (65, 40, 28672, 7), (100, 4096, 8192, 2),
    (128, 999, 32768, 8),
    # blocks of 128 x 128
    (130, 40, 16384, 8), (192, 4096, 8192, 4), (300, 1000, 10000, 4), (300, 4096, 8192, 2), (500, 600, 14336, 7),
    (1000, 100, 20480, 8)]


def _up(n, to):
    return -(-n // to) * to


def _splits(m, n, k, stride=None, x=FAKE):
    """How many workgroups share a block's inputs, from what the call's
    workspace holds beside codes and scales: a 4-byte ticket for each block of
    outputs and 8 bytes for each two sums of each split."""
    from mamba2_recall import _native
    need = _native.lib().m2r_int8_linear_workspace(x, k if stride is None else stride, m, n, k)
    rest = need - _up(_up(m, 16) * _up(k, 128), 256) - _up(4 * m, 256) if need else 0
    if rest == 0:
        return 1
    tiles = _up(m, 16) // 16
    if m <= 128:
        blocks, rows = _up(n, 32) // 32, next(t for t in (1, 2, 4, 8) if t >= tiles)
        part = 32 * 16 * rows * 4
    else:
        blocks, part = _up(m, 128) // 128 * (_up(n, 128) // 128), 128 * 128 * 4
    splits, left = divmod(rest - _up(4 * blocks, 256), blocks * part)
    assert left == 0
    return splits


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("m,n,k,splits", CASES)
def test_the_cases_are_split(m, n, k, splits, odd):
    assert _splits(m, n - odd, k) == splits


def _case(device, m, n, k, seed, dtype=F16):
    from mamba2_recall.int8 import Int8Weight
    gen = torch.Generator(device=device).manual_seed(seed)
    codes = torch.randint(-127, 128, (n, k), generator=gen, device=device, dtype=torch.int8)
    scale = (torch.rand(n, generator=gen, device=device) + 0.5) / 127 / k ** 0.5
    x = torch.randn(m, k, generator=gen, device=device).to(dtype)
    return x, codes, scale, Int8Weight(codes, scale)


def _formula(x, codes, scale):
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(127.0 * x / top).float()
    total = torch.zeros(x.shape[0], codes.shape[0], dtype=torch.float64, device=x.device)
    for i in range(0, x.shape[1], 1024):      # sums of 1,024 products are exact in binary32
        total += (q[:, i:i + 1024] @ codes[:, i:i + 1024].float().T).double()
    return total * (top / 127 * scale.double())


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("m,n,k,splits", CASES)
def test_split_products(device, m, n, k, splits, odd, dtype):
    from mamba2_recall.int8 import linear
    x, codes, scale, weight = _case(device, m, n - odd, k, m + n + k, F16 if odd else BF16)
    assert _splits(m, n - odd, k, x=x.data_ptr()) == splits
    want = _formula(x, codes, scale)
    # half a step of the type, five binary32 roundings, half a step of binary16's subnormals
    bound = want.abs() * (torch.finfo(dtype).eps / 2 + 5 * 2.0 ** -24) + 2.0 ** -25
    for _ in range(3):                        # tickets count from 0 in each call
        bad = ~((linear(x, weight, dtype).double() - want).abs() <= bound)
        assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


@gpu
def test_sums_at_the_ends_of_32_bits(device):
    """Partial sums and their total near 2^31, of both signs."""
    from mamba2_recall.int8 import Int8Weight, linear
    k = 131072
    codes = torch.full((40, k), 127, dtype=torch.int8, device=device)
    codes[1::3] = -128
    codes[2::3, 1::2] = -127
    scale = torch.full((40,), 2.0 ** -20, device=device)
    for m in (2, 20, 60, 100, 200):
        assert _splits(m, 40, k) == 8
        x = torch.ones(m, k, dtype=F16, device=device)
        x[1::2] = -1.0
        got = linear(x, Int8Weight(codes, scale), F32).double()
        total = torch.tensor([127.0 * 127 * k, -128.0 * 127 * k, 0.0], dtype=torch.float64, device=device).repeat(14)[:40]
        want = torch.where(torch.arange(m, device=device)[:, None] % 2 == 0, total, -total) * (2.0 ** -20 / 127)
        assert bool(((got - want).abs() <= want.abs() * 4 * 2.0 ** -24).all())   # sum, scale, two products


@gpu
@pytest.mark.parametrize("n,k", [(1000, 8192), (40, 32768)])
def test_split_and_unsplit_rows_are_equal(device, n, k):
    """A row's result does not depend on how many rows the call has, nor on how
    their inputs are split."""
    from mamba2_recall import int8
    x, _, _, weight = _case(device, 600, n, k, 3)
    spread = torch.empty(600, k + 1, dtype=F16, device=device)[:, 1:]   # no whole sixteens: codes in a launch of their own
    spread.copy_(x)
    whole, seen = int8.linear(x, weight), set()
    for lo, hi in ((0, 600), (0, 1), (1, 3), (3, 6), (6, 20), (20, 50), (50, 110), (110, 240), (240, 600)):
        assert torch.equal(int8.linear(x[lo:hi], weight), whole[lo:hi])
        assert torch.equal(int8.linear(spread[lo:hi], weight), whole[lo:hi])
        seen |= {_splits(hi - lo, n, k, x=x[lo:hi].data_ptr()), _splits(hi - lo, n, k, k + 1, spread[lo:hi].data_ptr())}
    # 40 channels of 32,768 inputs are split eight ways in every kernel; 8,192 inputs in one and more, as rows go
    assert seen == {8} if k == 32768 else {1} < seen


ROWS = (30, 64, 100, 300)


@gpu
@pytest.mark.parametrize("m", ROWS)
def test_graphs(device, m):
    """A captured split product, replayed with other inputs and with eager
    calls in between."""
    from mamba2_recall import int8
    x, _, _, weight = _case(device, m, 4096, 8192, m)
    assert _splits(m, 4096, 8192) > 1
    other, _, _, _ = _case(device, 77, 1, 8192, 99)
    int8.linear(x, weight)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = int8.linear(x, weight)
        second = int8.linear(x.neg(), weight)
    gen = torch.Generator(device=device).manual_seed(m)
    for _ in range(5):
        x.normal_(generator=gen)
        want = int8.linear(x, weight)
        int8.linear(other, weight)
        torch.cuda.synchronize()
        graph.replay()
        int8.linear(other, weight)
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, -want)


@gpu
def test_streams(device):
    """Split products on four streams at a time, each with tickets and sums of
    its own."""
    from mamba2_recall import int8
    rows = [_case(device, m, 1, 8192, m)[0] for m in ROWS]
    weight = _case(device, 1, 4096, 8192, 5)[3]
    assert all(_splits(m, 4096, 8192) > 1 for m in ROWS)
    want = [int8.linear(x, weight) for x in rows]
    streams = [torch.cuda.Stream() for _ in rows]
    torch.cuda.synchronize()
    got = [[] for _ in rows]
    for _ in range(8):
        for i, (x, s) in enumerate(zip(rows, streams)):
            with torch.cuda.stream(s):
                got[i].append(int8.linear(x, weight))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)
