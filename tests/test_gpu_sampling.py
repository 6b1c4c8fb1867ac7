"""Token sampling against the distribution in 64 bits.

Tolerance (derived): a weight 2^-d, d < 32, has its exponent computed by a
subtraction and a product in binary32 (3 roundings of a rate and an exponent
of at most 32: 32 * 3 * 2^-24 * ln 2) and its power rounded to 2^-23, so that
weights, their sums and the shares of the row are within EPS = 8e-6 of the
64-bit ones, relatively; weights below 2^-31 of the largest are dropped
(V 2^-31 of the whole at most).  The drawn token's interval of the
distribution function then holds the given number to 2 EPS + V 2^-31, and its
place in the sorted row satisfies the filters to the same.  Where all weights
are equal the arithmetic is exact, and so are the tests."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 8e-6
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _logits(device, batch, vocab, dtype, seed, spread=2.5):
    gen = torch.Generator(device=device).manual_seed(seed)
    l = torch.randn(batch, vocab, generator=gen, device=device) * spread
    return l.to(dtype), torch.rand(batch, generator=gen, device=device)


def _verify(logits, uniforms, ids, logprobs, temperature, top_k, top_p, min_p):
    """Every row's token against the distribution in float64."""
    batch, vocab = logits.shape
    slack = 2 * EPS + vocab * 2.0 ** -31

    def row(v, b):
        return float(v[b]) if isinstance(v, torch.Tensor) else float(v)
    for b in range(batch):
        l = torch.nan_to_num(logits[b].double().cpu(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        token, t, k = int(ids[b]), row(temperature, b), int(row(top_k, b))
        if t <= 0:
            t, k = 1.0, 1
        w = torch.exp((l - l.max()) / t)
        order = torch.sort(l, descending=True, stable=True).indices
        n = min(k, vocab) if k > 0 else vocab
        place = int((order == token).nonzero())
        assert place < n, f"row {b}: token outside top-k"
        ws = w[order][:n] / w[order][:n].sum()
        cum = torch.cumsum(ws, 0)
        p = row(top_p, b)
        before = float(cum[place] - ws[place])
        assert place == 0 or p >= 1 or before <= p + slack, f"row {b}: token outside top-p"
        assert place == 0 or float(w[token]) >= row(min_p, b) * (1 - slack), f"row {b}: token outside min-p"
        # the kept sets that rounding at a filter's edge allows: smallest and largest
        keep = []
        for edge in (-slack, slack):
            m = n if p >= 1 else min(n, int((cum - ws < p + edge).sum()))
            m = min(m, int((w[order] >= row(min_p, b) * (1 - edge)).sum()))
            mask = torch.zeros(vocab, dtype=torch.bool)
            mask[order[:max(1, m)]] = True
            keep.append(torch.where(mask, w, 0.0))
        u, ok = float(uniforms[b]), False
        lows, highs, lps = [], [], []
        for kept in keep:
            total = kept.sum()
            hi = float(kept[:token + 1].sum() / total)
            lows.append(hi - float(kept[token] / total))
            highs.append(hi)
            lps.append(float(torch.log(w[token] / total)))
        assert min(lows) - slack <= u <= max(highs) + slack, f"row {b}: token {token} not at {u}: {lows} {highs}"
        got = float(logprobs[b])
        tol = slack + 2.0 ** -22 * max(1.0, abs(got)) + abs(lps[0] - lps[1])
        assert abs(got - lps[0]) <= tol, f"row {b}: log probability {got}, {lps}"


def _sample(logits, uniforms, **kw):
    from mamba2_recall import sampling
    return sampling.sample(logits, uniforms, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4097, 50003])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.7, top_k=50, top_p=0.9), dict(top_p=0.8),
                                dict(top_k=5), dict(min_p=0.05), dict(temperature=1.5, top_k=3000, top_p=0.99, min_p=1e-3),
                                dict(temperature=0.0)])
def test_filters(device, dtype, vocab, kw):
    logits, u = _logits(device, 6, vocab, dtype, seed=vocab)
    ids, lp = _sample(logits, u, **kw)
    full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    full.update(kw)
    _verify(logits, u, ids, lp, **full)


@pytest.mark.parametrize("vocab", [256000, 131072])
def test_large_rows_with_filters_of_their_own(device, vocab):
    logits, u = _logits(device, 12, vocab, torch.float16, seed=1)

    def each(values, dtype):
        return torch.tensor(values, dtype=dtype, device=device)
    kw = dict(temperature=each([1, 0, 0.5, 1, 1, 2, 0.8, 1, 1, 1, 0.1, 5], torch.float32),
              top_k=each([0, 7, 0, 50, 0, 0, 1, 20000, 200000, 2 ** 31 - 1, -4, 1000], torch.int32),
              top_p=each([1, 1, 0.9, 1, 0.999, 0.5, 1, 0.7, 0.9, 1, 0.0, 0.95], torch.float32),
              min_p=each([0, 0, 0, 0.3, 0, 1e-4, 0, 0, 0, 0.02, 0, 1], torch.float32))
    ids, lp = _sample(logits, u, **kw)
    _verify(logits, u, ids, lp, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spread", [0.02, 1e-3, 1.0, 60.0])
@pytest.mark.parametrize("masked", [None, "lowest", "inf", "far"])
def test_close_and_distant_logits(device, dtype, spread, masked):
    """Logits that nearly all weigh the same, or nearly nothing; a mask's
    finite value tells nothing about the others' range."""
    logits, u = _logits(device, 4, 100001, dtype, seed=7, spread=spread)
    if masked:
        value = {"lowest": torch.finfo(dtype).min, "inf": -math.inf, "far": float(logits.float().min()) - 25.0}[masked]
        logits[:, ::3] = value
        logits[0, :99000] = value
    for kw in (dict(top_p=0.9), dict(top_k=50), dict(top_k=5000, top_p=0.9), dict(temperature=0.0),
               dict(temperature=3.0, top_p=0.3)):
        ids, lp = _sample(logits, u, **kw)
        full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
        full.update(kw)
        _verify(logits, u, ids, lp, **full)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [5, 4096, 100001])
def test_equal_logits_exactly(device, dtype, vocab):
    """All weights equal: the token is floor(u n) of the first n kept ones."""
    logits = torch.full((5, vocab), -3.25, dtype=dtype, device=device)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24], device=device)
    one = 2 ** 31

    def token(x, n):
        return min(int(math.floor(float(x) * float(n * one))), n * one - 1) // one
    for kw, n in ((dict(), vocab), (dict(top_k=3), 3), (dict(top_k=3000), min(vocab, 3000)),
                  (dict(top_p=0.5), -(-vocab // 2)), (dict(min_p=1.0), vocab), (dict(temperature=0.0), 1),
                  (dict(top_k=4, top_p=0.5), 2), (dict(top_p=0.0), 1)):
        ids, lp = _sample(logits, u, **kw)
        assert ids.tolist() == [token(x, n) for x in u], (kw, n)
        assert torch.allclose(lp.double().cpu(), torch.full((5,), -math.log(n), dtype=torch.float64), atol=1e-6, rtol=1e-6)


@pytest.mark.parametrize("values", [[0.5, 0.25], [0.0, -0.0, 3.0, -1.0], [1.0, 1.0009765625, 1.001953125, 0.5, -30.0]])
@pytest.mark.parametrize("vocab", [30000, 100001])
def test_few_values_among_many_tokens(device, values, vocab):
    """Thousands of tokens of each logit: more than a list holds, cut inside
    one value's tokens by count and by weight."""
    gen = torch.Generator(device=device).manual_seed(vocab)
    pick = torch.randint(0, len(values), (5, vocab), generator=gen, device=device)
    logits = torch.tensor(values, device=device)[pick]
    u = torch.rand(5, generator=gen, device=device)
    for kw in (dict(top_k=7000), dict(top_k=vocab - 3), dict(top_p=0.37), dict(top_k=9999, top_p=0.8, min_p=0.3),
               dict(temperature=0.0), dict(temperature=0.02, top_p=0.5)):
        ids, lp = _sample(logits, u, **kw)
        full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
        full.update(kw)
        _verify(logits, u, ids, lp, **full)


def test_ties_go_to_the_lowest_index(device):
    logits = torch.full((3, 9000), -8.0, dtype=torch.float16, device=device)
    logits[:, [17, 4000, 8000, 8999]] = 4.0
    logits[:, 6000] = 4.5
    u = torch.tensor([0.0, 0.5, 0.999], device=device)
    assert _sample(logits, u, temperature=0.0)[0].tolist() == [6000] * 3
    # the first two of the four equal ones stay: shares 0.274, 0.274, 0.452
    assert _sample(logits, u, top_k=3)[0].tolist() == [17, 4000, 6000]
    logits[:, 6000] = -8.0
    assert _sample(logits, u, top_k=2)[0].tolist() == [17, 4000, 4000]
    assert _sample(logits, u, temperature=0.0)[0].tolist() == [17] * 3
    # zeros of either sign are equal
    zeros = torch.full((3, 100), -5.0, device=device)
    zeros[:, 40], zeros[:, 50] = -0.0, 0.0
    assert _sample(zeros, u, top_k=1)[0].tolist() == [40] * 3
    # nothing but ties above the cut, more of them than a workgroup has threads
    many = torch.full((3, 20000), -1.0, device=device)
    many[:, 5000:] = 1.0
    assert _sample(many, u, top_k=6000)[0].tolist() == [5000, 8000, 5000 + int(0.999 * 6000)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_tokens(device, dtype):
    """-inf, the type's lowest value, NaN and +inf; a row with nothing left."""
    logits, u = _logits(device, 6, 5000, dtype, seed=3)
    low = torch.finfo(dtype).min
    logits[0, 10:] = -math.inf
    logits[1, 10:] = low
    logits[2, 10:] = math.nan
    logits[3] = -math.inf
    logits[4] = math.nan
    logits[5, [70, 90]] = math.inf
    for kw in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(temperature=0.0), dict(temperature=100.0)):
        ids, lp = _sample(logits, u, **kw)
        assert all(0 <= int(ids[b]) < 10 for b in range(3)), kw
        assert ids[3:5].tolist() == [-1, -1] and bool((lp[3:5] == -math.inf).all())
        assert int(ids[5]) in (70, 90)
    lowest = torch.full((2, 300), low, dtype=dtype, device=device)   # equal, so all as likely
    assert _sample(lowest, torch.tensor([0.0, 0.5], device=device))[0].tolist() == [0, 150]
    ends = torch.full((2, 300), low, dtype=dtype, device=device)
    ends[:, 123] = torch.finfo(dtype).max
    assert _sample(ends, torch.tensor([0.0, 0.999], device=device), top_p=0.9)[0].tolist() == [123, 123]


def test_uniform_ends(device):
    """Numbers outside [0, 1) draw the nearest end, not outside the row."""
    logits = torch.zeros(5, 1000, device=device)
    u = torch.tensor([0.0, 1.0, -1.0, 7.0, math.nan], device=device)
    assert _sample(logits, u)[0].tolist() == [0, 999, 0, 999, 0]


def test_distribution(device):
    """Draws over a grid of given numbers: every token its share of them."""
    logits, _ = _logits(device, 1, 40, torch.float32, seed=8, spread=1.0)
    n = 4096
    u = (torch.arange(n, device=device) + 0.5) / n
    ids, _ = _sample(logits.expand(n, 40).contiguous(), u, top_k=30, top_p=0.95)
    share = torch.bincount(ids.cpu(), minlength=40).double() / n
    p = torch.softmax(logits[0].double().cpu(), 0)
    order = torch.sort(p, descending=True).indices
    head = p[order[:30]] / p[order[:30]].sum()
    m = int((torch.cumsum(head, 0) - head < 0.95).sum())
    want = torch.zeros(40, dtype=torch.float64)
    want[order[:m]] = p[order[:m]] / p[order[:m]].sum()
    assert float((share - want).abs().max()) <= 1.0 / n + 2 * EPS


def test_rows_alone_or_together(device):
    """A row's result depends on neither its neighbours nor its place."""
    logits, u = _logits(device, 40, 30011, torch.float16, seed=9)
    kw = dict(temperature=0.9, top_k=300, top_p=0.97)
    ids, lp = _sample(logits, u, **kw)
    for b in (0, 7, 39):
        one = _sample(logits[b:b + 1], u[b:b + 1], **kw)
        assert int(one[0]) == int(ids[b]) and float(one[1]) == float(lp[b])
    again = _sample(logits, u, **kw)
    assert torch.equal(again[0], ids) and torch.equal(again[1], lp)
    wide = torch.full((40, 30020), 50.0, dtype=torch.float16, device=device)
    wide[:, 3:30014] = logits
    view = _sample(wide[:, 3:30014], u, **kw)
    assert torch.equal(view[0], ids) and torch.equal(view[1], lp)
    turned = _sample(logits.t().contiguous().t(), u, **kw)
    assert torch.equal(turned[0], ids)


@pytest.mark.parametrize("batch", [2, 30])
def test_stream_and_graph(device, batch):
    from mamba2_recall import sampling
    logits, u = _logits(device, batch, 20000, torch.float16, seed=10)
    kw = dict(top_k=40, top_p=0.9)
    want = _sample(logits, u, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _sample(logits, u, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampling.sample(logits, u, **kw)
    for seed in range(3):
        fresh, fu = _logits(device, batch, 20000, torch.float16, seed=20 + seed)
        logits.copy_(fresh)
        u.copy_(fu)
        graph.replay()
        want = _sample(logits, u, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals(device):
    logits, u = _logits(device, 3, 100, torch.float16, seed=1)
    bad = [(logits[0], u, {}), (logits.double(), u, {}), (logits.cpu(), u.cpu(), {}), (logits, u[:2], {}),
           (logits, u.half(), {}), (logits, u.cpu(), {}), (logits[:, :0], u, {}),
           (logits, u, dict(temperature=-1.0)), (logits, u, dict(temperature=math.nan)), (logits, u, dict(top_k=-1)),
           (logits, u, dict(top_k=2.0)), (logits, u, dict(top_p=1.5)), (logits, u, dict(min_p=-0.1)),
           (logits, u, dict(top_k=torch.zeros(3, device=device))), (logits, u, dict(top_p=torch.ones(2, device=device))),
           (logits, u, dict(min_p=torch.zeros(3)))]
    for l, x, kw in bad:
        with pytest.raises(ValueError):
            _sample(l, x, **kw)
    ids, lp = _sample(logits[:0], u[:0])
    assert ids.shape == (0,) and lp.shape == (0,)
