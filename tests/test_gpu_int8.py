"""Projections in 8-bit integers (int8.linear, Int8Weight) against the formula
in whole numbers and binary64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rows(device, m, k, dtype, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(m, k, generator=gen, device=device) * (torch.rand(m, 1, generator=gen, device=device) * 3 + 0.01)
    x[:, torch.randint(0, k, (1 + k // 300,), generator=gen, device=device)] *= 9.0
    return x.to(dtype)


def _weight(device, n, k, seed):
    from mamba2_recall.int8 import Int8Weight
    gen = torch.Generator(device=device).manual_seed(seed)
    codes = torch.randint(-127, 128, (n, k), generator=gen, device=device, dtype=torch.int8)
    scale = (torch.rand(n, generator=gen, device=device) + 0.5) / 127 / k ** 0.5
    return codes, scale, Int8Weight(codes, scale)


def _codes(x):
    """rint(127 x / max|x|) as in exact arithmetic: the quotient in binary64 is
    not within 2^-19 of a tie unless it is one, which binary64 holds."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    return torch.where(top > 0, torch.round(127.0 * x / top), torch.zeros_like(x)), top[:, 0]


def _check(x, codes, scale, weight, dtype):
    from mamba2_recall import int8
    y = int8.linear(x, weight, dtype)
    assert y.dtype == (dtype or x.dtype) and y.shape == (*x.shape[:-1], codes.shape[0])
    q, top = _codes(x.reshape(-1, x.shape[-1]).cpu())
    want = q @ codes.double().cpu().T
    assert float(want.abs().max()) < 2 ** 31
    want = want * (top[:, None] / 127 * scale.double().cpu())
    # the type's half step; five binary32 roundings (scale, sum, two products, one more for the weights' scale), the
    # scale's being 2^-150 at least, half a step of binary32's subnormals; half a step of the type's
    step = 2.0 ** -150 / (top[:, None] / 127).clamp(min=2.0 ** -150)
    least = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps / 2
    bound = want.abs() * (torch.finfo(y.dtype).eps / 2 + 5 * 2.0 ** -24 + step) + least
    got = y.double().cpu().reshape(want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:5].tolist(), got[bad][:5], want[bad][:5])
    return y


SIZES = [(1, 1, 1), (1, 16, 64), (2, 17, 65), (3, 5, 200), (15, 40, 127), (16, 64, 128), (17, 33, 129), (5, 300, 1000),
         (33, 250, 320), (64, 128, 512), (65, 130, 640), (77, 2041, 1000), (100, 100, 100), (128, 256, 256),
         (129, 257, 385), (200, 1000, 96), (255, 255, 255), (256, 512, 1024), (257, 520, 2048), (300, 48, 4096),
         (513, 777, 640), (1000, 300, 300)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("x_dtype,dtype", [(F16, None), (BF16, F32), (F16, BF16)])
def test_sizes(device, m, n, k, x_dtype, dtype):
    codes, scale, weight = _weight(device, n, k, m + n)
    _check(_rows(device, m, k, x_dtype, k), codes, scale, weight, dtype)


@pytest.mark.parametrize("m", list(range(1, 20)) + [24, 31, 32, 47, 48, 49, 63, 79, 95, 96, 97, 111, 127, 160, 191, 192, 193])
def test_rows(device, m):
    codes, scale, weight = _weight(device, 150, 700, m)
    _check(_rows(device, m, 700, F16, m), codes, scale, weight, F32)


@pytest.mark.parametrize("m,n,k", [(1, 18560, 4096), (4, 4096, 8192), (16, 18560, 4096), (64, 4096, 8192),
                                   (70, 18560, 4096), (300, 4096, 8192), (600, 4096, 4096)])
def test_projections(device, m, n, k):
    codes, scale, weight = _weight(device, n, k, m)
    _check(_rows(device, m, k, F16, m), codes, scale, weight, None)


def test_head(device):
    codes, scale, weight = _weight(device, 256000, 256, 1)
    for m in (1, 24):
        _check(_rows(device, m, 256, F16, m), codes, scale, weight, F32)


def test_rows_do_not_depend_on_the_batch(device):
    from mamba2_recall import int8
    _, _, weight = _weight(device, 1000, 900, 3)
    x = _rows(device, 600, 900, F16, 4)
    whole = int8.linear(x, weight)
    for lo, hi in ((0, 1), (1, 3), (3, 20), (20, 60), (60, 190), (190, 600)):
        assert torch.equal(int8.linear(x[lo:hi], weight), whole[lo:hi])


def test_longest_inputs(device):
    """Sums at the ends of 32 bits."""
    from mamba2_recall.int8 import Int8Weight
    k = 131072
    codes = torch.full((20, k), 127, dtype=torch.int8, device=device)
    codes[1] = -128
    codes[2, 1::2] = -127
    x = torch.ones(3, k, dtype=F16, device=device)
    x[1] = -1.0
    x[2, ::3] = 0.25
    scale = torch.full((20,), 1e-5, device=device)
    y = _check(x, codes, scale, Int8Weight(codes, scale), F32)
    assert float(y[0, 2]) == 0.0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_codes_of_every_quotient(device, dtype):
    """All values against largest values over the whole range, ties among them:
    the codes are those of exact arithmetic, the scales binary32's nearest."""
    from mamba2_recall.int8 import Int8Weight
    every = torch.arange(0x7c00 if dtype == F16 else 0x7f80, dtype=torch.int32).to(torch.int16).view(dtype).to(device)
    limit = every.numel()
    gen = torch.Generator().manual_seed(1)
    tops = torch.cat((torch.tensor([0, 1, 2, 3, 127, 254, 255, 0x3ff, limit - 1, limit - 2]),
                      torch.randint(1, limit, (300,), generator=gen)))
    if dtype == F16:      # largest values whose quotients have many ties: multiples of 127 and 254
        tops = torch.cat((tops, torch.tensor([float(127 * i) for i in range(1, 300)]).half().view(torch.int16).long(),
                          torch.tensor([127 * i / 16 for i in range(1, 128)]).half().view(torch.int16).long()))
    for part in tops.split(64):
        top = every[part.to(device)]
        x = torch.where(every <= top[:, None], every, torch.zeros_like(every))     # the largest is among them
        x = torch.cat((x, -x), 1) if x.shape[1] * 2 <= 131072 else x
        w = Int8Weight.quantize(x.contiguous())
        want, largest = _codes(x)
        assert torch.equal(w.codes.double(), want)
        # binary64's quotient rounded again is binary32's nearest: 127 does not divide a number of 11 bits
        # to within 2^-30 of a point halfway between two of binary32's
        assert torch.equal(w.scale, (largest / 127.0).float())


def test_quantized_weights(device):
    from mamba2_recall import int8
    for dtype in (F16, BF16):
        w = _rows(device, 100, 333, dtype, 5)
        q = int8.Int8Weight.quantize(w)
        again = int8.Int8Weight(q.codes, q.scale)
        assert q.features == (333, 100) and torch.equal(again.tiles, q.tiles)
        want, top = _codes(w)
        assert torch.equal(q.codes.double(), want)
        # a code is off by at most half a step of its channel; the scale and the product are rounded to binary32,
        # two halves of 2^-23 of at most 127 steps: 127 * 2^-23 < 2^-16 of a step, 2^-15 of half a step
        assert bool(((q.decode(F32).double() - w.double()).abs() <= (top[:, None] / 254) * (1 + 2.0 ** -15)).all())
        wide = torch.zeros(100, 700, dtype=dtype, device=device)
        for view in (wide[:, 7:340], wide[:, 1:667:2]):
            view.copy_(w)
            assert torch.equal(int8.Int8Weight.quantize(view).tiles, q.tiles)
        x = _rows(device, 9, 333, dtype, 6)
        assert torch.equal(q(x, F32), int8.linear(x, q, F32))


def test_views(device):
    from mamba2_recall import int8
    codes, scale, weight = _weight(device, 90, 260, 7)
    x = _rows(device, 24, 260, F16, 8)
    want = _check(x, codes, scale, weight, None)
    wide = torch.zeros(24, 901, dtype=F16, device=device)
    for view in (wide[:, 3:263], wide[:, 1:521:2]):
        view.copy_(x)
        assert torch.equal(int8.linear(view, weight), want)
    assert torch.equal(int8.linear(x.view(2, 3, 4, 260), weight), want.view(2, 3, 4, 90))
    assert torch.equal(int8.linear(x[5], weight), want[5])
    assert torch.equal(int8.linear(x[:1].expand(6, -1), weight), want[:1].expand(6, -1))
    assert torch.equal(int8.linear(x.view(4, 6, 260).transpose(0, 1), weight), want.view(4, 6, 90).transpose(0, 1))
    assert int8.linear(x[:0], weight).shape == (0, 90)
    spread = int8.Int8Weight(codes.t().contiguous().t(), scale.repeat_interleave(2)[::2])
    assert torch.equal(int8.linear(x, spread), want)


@pytest.mark.parametrize("m", [1, 7, 40, 200])
def test_rows_that_are_not_finite_and_rows_of_zeros(device, m):
    from mamba2_recall import int8
    for dtype in (F16, BF16):
        _, _, weight = _weight(device, 70, 500, 9)
        x = _rows(device, m, 500, dtype, 10)
        want = int8.linear(x, weight)
        for bad in (float("nan"), float("inf"), float("-inf")):
            y = x.clone()
            y[m // 2, 499] = bad
            got = int8.linear(y, weight)
            assert bool(torch.isnan(got[m // 2]).all())
            keep = torch.arange(m, device=device) != m // 2
            assert torch.equal(got[keep], want[keep])
        y = x.clone()
        y[m // 2] = 0.0
        got = int8.linear(y, weight)
        assert not bool(got[m // 2].any())


def test_scales_at_the_ends_of_their_range(device):
    """Values near the types' largest and least: no product on the way leaves
    binary32's range while the result is in it."""
    from mamba2_recall.int8 import Int8Weight
    gen = torch.Generator(device=device).manual_seed(11)
    codes = torch.randint(-127, 128, (50, 300), generator=gen, device=device, dtype=torch.int8)
    for x_scale, w_scale in ((1e30, 1e-34), (1e-30, 1e32), (1e-36, 1e36), (1e36, 1e-37), (2.0 ** -130, 2.0 ** 120)):
        x = (torch.randn(40, 300, generator=gen, device=device).double() * x_scale).to(BF16)
        x[3] = 0
        scale = torch.full((50,), w_scale, device=device)
        _check(x, codes, scale, Int8Weight(codes, scale), F32)
    x = torch.tensor([[65504.0, -65504.0, 6e-8, 2.0]], device=device).half()
    codes = torch.tensor([[127, -128, 3, 4], [0, 0, 127, 0]], dtype=torch.int8, device=device)
    scale = torch.tensor([1e-3, 1.0], device=device)
    _check(x, codes, scale, Int8Weight(codes, scale), F32)


def test_other_stream_and_graph(device):
    from mamba2_recall import int8
    _, _, weight = _weight(device, 4096, 2048, 12)
    for m in (1, 30, 400):
        x = _rows(device, m, 2048, F16, 13)
        want = int8.linear(x, weight)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            side = int8.linear(x, weight)
        stream.synchronize()
        assert torch.equal(side, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = int8.linear(x, weight)
        for step in range(4):
            x.copy_(_rows(device, m, 2048, F16, 20 + step))
            want = int8.linear(x, weight)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_two_calls_at_once(device):
    """Calls on two streams, each with workspaces of its own."""
    from mamba2_recall import int8
    _, _, weight = _weight(device, 4096, 1024, 14)
    rows = [_rows(device, m, 1024, F16, m) for m in (3, 64, 130, 500)]
    want = [int8.linear(x, weight) for x in rows]
    streams = [torch.cuda.Stream() for _ in rows]
    torch.cuda.synchronize()
    got = [[] for _ in rows]
    for _ in range(5):
        for i, (x, s) in enumerate(zip(rows, streams)):
            with torch.cuda.stream(s):
                got[i].append(int8.linear(x, weight))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)


def test_refusals(device):
    from mamba2_recall import int8
    _, _, weight = _weight(device, 8, 16, 15)
    x = _rows(device, 2, 16, F16, 16)
    for bad in (x.float(), x[:, :15], x.cpu(), None, x.new_zeros(())):
        with pytest.raises(ValueError):
            int8.linear(bad, weight)
    for kw in (dict(dtype=torch.int8), dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            int8.linear(x, weight, **kw)
    with pytest.raises(ValueError):
        int8.linear(x, x)
    codes = torch.zeros(4, 16, dtype=torch.int8, device=device)
    for args in ((codes.short(), torch.ones(4, device=device)), (codes, torch.ones(3, device=device)),
                 (codes, torch.ones(4)), (codes[0], torch.ones(16, device=device)), (codes, torch.ones(4, device=device).half()),
                 (codes[:0], torch.ones(0, device=device)),
                 (torch.zeros(1, 131073, dtype=torch.int8, device=device), torch.ones(1, device=device))):
        with pytest.raises(ValueError):
            int8.Int8Weight(*args)
    for bad in (x.float(), x[0], x.cpu(), x[:0]):
        with pytest.raises(ValueError):
            int8.Int8Weight.quantize(bad)


def test_offsets_past_32_bits(device):
    """More than 2^31 outputs, codes and weights: the last rows and channels are
    those of small calls."""
    from mamba2_recall import int8
    gen = torch.Generator(device=device).manual_seed(17)
    codes, scale, weight = _weight(device, 256000, 64, 18)
    x = torch.randn(8500, 64, generator=gen, device=device).half()
    y = int8.linear(x, weight)
    assert torch.equal(y[-5:], int8.linear(x[-5:], weight)) and torch.equal(y[:5], int8.linear(x[:5], weight))
    del y
    _, _, weight = _weight(device, 40, 4096, 19)
    x = torch.empty(600001, 4096, dtype=F16, device=device).normal_(generator=gen)
    y = int8.linear(x, weight)
    assert torch.equal(y[-70:], int8.linear(x[-70:], weight)) and torch.equal(y[:3], int8.linear(x[:3], weight))
    del x, y
    codes = torch.empty(600001, 4096, dtype=torch.int8, device=device).random_(-127, 128, generator=gen)
    scale = torch.rand(600001, generator=gen, device=device) * 1e-4
    weight, tail = int8.Int8Weight(codes, scale), int8.Int8Weight(codes[-33:], scale[-33:])
    del codes
    for m in (2, 30, 140):
        x = _rows(device, m, 4096, F16, m)
        assert torch.equal(int8.linear(x, weight)[:, -33:], int8.linear(x, tail))
