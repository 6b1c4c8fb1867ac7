"""Penalties, biases and masks on logits (sampling.adjust) against the formula
in binary64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


def _row(value, i):
    return float(value[i]) if isinstance(value, torch.Tensor) else float(torch.tensor(value, dtype=torch.float32))


def _oracle(logits, prompt=None, prompt_lengths=None, tokens=None, lengths=None, repetition=1.0, presence=0.0,
            frequency=0.0, bias=None, allowed=None, allowed_rows=None):
    """(logits in binary64, the magnitudes that were added up, where they were touched) on the host, token by token."""
    l = logits.double().cpu().clone()
    batch, vocab = l.shape
    size, touched = l.abs().clone(), torch.zeros(batch, vocab, dtype=torch.bool)

    def ids(t, n, i):
        if t is None:
            return []
        n = t.shape[1] if n is None else max(0, min(t.shape[1], int(n[i])))
        return [v for v in t[i, :n].tolist() if 0 <= v < vocab]
    for i in range(batch):
        new, old = ids(tokens, lengths, i), ids(prompt, prompt_lengths, i)
        r, p, f = _row(repetition, i), _row(presence, i), _row(frequency, i)
        counts = {}
        for v in new:
            counts[v] = counts.get(v, 0) + 1
        for v in set(new) | set(old):
            x = float(l[i, v])
            x = x / r if x > 0 else x * r
            size[i, v] = max(abs(x), float(size[i, v]))
            c = counts.get(v, 0)
            if c:
                x -= f * c + p
                size[i, v] += abs(f) * c + abs(p)
            l[i, v] = x
            touched[i, v] = True
        if bias is not None:
            b_ids, values = bias
            last = {}
            for v, x in zip((b_ids if b_ids.ndim == 1 else b_ids[i]).tolist(),
                            (values if values.ndim == 1 else values[i]).tolist()):
                last[v] = x
            for v, x in last.items():
                if 0 <= v < vocab:
                    l[i, v] += x
                    size[i, v] += abs(x)
                    touched[i, v] = True
        if allowed is not None:
            m = 0 if allowed.ndim == 1 else (i if allowed_rows is None else int(allowed_rows[i]))
            rows = allowed[None] if allowed.ndim == 1 else allowed
            if 0 <= m < rows.shape[0]:
                words = rows[m].long().cpu() & 0xffffffff
                free = (words[:, None] >> torch.arange(32) & 1).flatten()[:vocab].bool()
                l[i, ~free] = -INF
                touched[i, ~free] = True
    return l, size, touched


def _check(logits, **kw):
    from mamba2_recall import sampling
    want, size, touched = _oracle(logits, **kw)
    before = logits.clone()
    got = sampling.adjust(logits, **kw)
    assert got.dtype == logits.dtype and got.is_contiguous() and torch.equal(_bits(logits), _bits(before))
    assert torch.equal(_bits(got).cpu()[~touched], _bits(logits).cpu()[~touched])
    # half a step of the type; five binary32 roundings of values no larger than `size`; binary16's subnormals
    bound = (want.abs() * (torch.finfo(logits.dtype).eps / 2) + 5 * 2.0 ** -24 * size
             + (2.0 ** -25 if logits.dtype == torch.float16 else 0.0))
    limit = torch.finfo(logits.dtype).max
    g = got.double().cpu()
    same = (g == want) | (torch.isnan(g) & torch.isnan(want)) | (torch.isinf(g) & (want.abs() > limit * (1 - 2.0 ** -9))
                                                                & (torch.sign(g) == torch.sign(want)))
    bad = touched & ~same & ~((g - want).abs() <= bound)
    assert not bool(bad.any()), (bad.nonzero()[:4].tolist(), g[bad][:4], want[bad][:4])
    # into the logits themselves, and into memory of another stride: the same bits
    place = logits.clone()
    assert sampling.adjust(place, out=place, **kw) is place and torch.equal(_bits(place), _bits(got))
    apart = torch.empty(logits.shape[0], logits.shape[1] + 5, dtype=logits.dtype, device=logits.device)[:, 3:-2]
    assert torch.equal(_bits(sampling.adjust(logits, out=apart, **kw)), _bits(got))
    return got


def _bits(t):
    return t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)


def _case(device, dtype, batch, vocab, prompt, tokens, bias, masks, seed=0, wide=True):
    gen = torch.Generator(device=device).manual_seed(seed)

    def ids(n):   # a third in a few tokens, some outside the vocabulary
        t = torch.randint(-2, vocab + 3, (batch, n), generator=gen, device=device)
        few = torch.randint(0, min(vocab, 5), (batch, n), generator=gen, device=device)
        t = torch.where(torch.rand(batch, n, generator=gen, device=device) < 0.3, few, t)
        return t if wide else t.to(torch.int32)

    def rows(low, high):
        return torch.rand(batch, generator=gen, device=device) * (high - low) + low
    kw = dict(repetition=rows(0.7, 1.6), presence=rows(-1, 1), frequency=rows(-0.3, 0.5))
    if prompt:
        kw.update(prompt=ids(prompt), prompt_lengths=torch.randint(-1, prompt + 2, (batch,), generator=gen, device=device,
                                                                   dtype=torch.int32))
    if tokens:
        kw.update(tokens=ids(tokens), lengths=torch.randint(-1, tokens + 2, (batch,), generator=gen, device=device,
                                                            dtype=torch.int32))
    if bias:
        kw["bias"] = (torch.randint(-2, vocab + 2, (batch, bias), generator=gen, device=device, dtype=torch.int32),
                      torch.randn(batch, bias, generator=gen, device=device) * 4)
    if masks:
        words = (vocab + 31) // 32
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (masks, words), generator=gen, device=device).to(torch.int32)
        kw["allowed"][0] = 0      # a mask that leaves nothing
        kw["allowed_rows"] = torch.randint(-1, masks + 1, (batch,), generator=gen, device=device, dtype=torch.int32)
    logits = (torch.randn(batch, vocab, generator=gen, device=device) * 4).to(dtype)
    return logits, kw


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 1000, 4095, 4096, 4097, 20001])
def test_sizes(device, dtype, vocab):
    logits, kw = _case(device, dtype, 3, vocab, 37, 21, 9, 2, seed=vocab)
    _check(logits, **kw)


@pytest.mark.parametrize("prompt,tokens,bias,masks,wide", [
    (0, 0, 0, 0, True), (1, 0, 0, 0, True), (0, 1, 0, 0, False), (0, 0, 1, 0, True), (0, 0, 0, 3, True),
    (5000, 0, 0, 0, False), (0, 3001, 0, 0, True), (2000, 700, 0, 0, True), (2000, 700, 300, 0, False),
    (0, 0, 300, 5, True), (2000, 700, 1200, 7, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_parts(device, dtype, prompt, tokens, bias, masks, wide):
    logits, kw = _case(device, dtype, 5, 9001, prompt, tokens, bias, masks, seed=prompt + tokens, wide=wide)
    _check(logits, **kw)


@pytest.mark.parametrize("batch", [1, 2, 17, 300])
def test_rows(device, batch):
    logits, kw = _case(device, torch.bfloat16, batch, 777, 50, 20, 5, 4, seed=batch)
    _check(logits, **kw)


def test_large_vocabularies(device):
    for batch, vocab in ((2, 256000), (1, 600001)):
        logits, kw = _case(device, torch.float32, batch, vocab, 3000, 900, 100, 2, seed=vocab)
        _check(logits, **kw)


def test_numbers_and_defaults(device):
    logits, kw = _case(device, torch.float16, 4, 3000, 60, 60, 0, 0, seed=3)
    kw.update(repetition=1.3, presence=0.5, frequency=0.25)
    kw.pop("lengths"), kw.pop("prompt_lengths")
    _check(logits, **kw)
    from mamba2_recall import sampling
    same = sampling.adjust(logits)
    assert torch.equal(_bits(same), _bits(logits)) and same.data_ptr() != logits.data_ptr()
    # settings of 1 and 0 change nothing, whatever the ids
    assert torch.equal(sampling.adjust(logits, prompt=kw["prompt"], tokens=kw["tokens"]), logits)
    assert sampling.adjust(logits[:0]).shape == (0, 3000)


def test_one_bias_and_one_mask_for_all_rows(device):
    from mamba2_recall import sampling
    logits, _ = _case(device, torch.float32, 3, 100, 0, 0, 0, 0, seed=4)
    ids = torch.tensor([7, 3, 7, -1, 100, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=device)
    values = torch.tensor([1.0, 2.0, -5.0, 9.0, 9.0, 9.0, 9.0], device=device)
    mask = torch.tensor([-1, 0, 5, 15], dtype=torch.int32, device=device)
    got = _check(logits, bias=(ids, values), allowed=mask)
    assert torch.equal(got[:, 7], logits[:, 7] - 5.0)       # the later entry of token 7
    assert bool(torch.isinf(got[:, 32:64]).all())
    per_row = sampling.adjust(logits, bias=(ids.expand(3, -1), values.expand(3, -1)), allowed=mask.expand(3, -1))
    assert torch.equal(per_row, got)


def test_ids_beyond_32_bits(device):
    """An int64 id whose low half is a token's is not that token."""
    logits, _ = _case(device, torch.float32, 1, 50, 0, 0, 0, 0, seed=5)
    ids = torch.tensor([[2 ** 32 + 3, 2 ** 40, -2 ** 62, -1, 49, 50]], device=device)
    _check(logits, tokens=ids, presence=1.0, repetition=2.0)


def test_views(device):
    logits, kw = _case(device, torch.float16, 4, 501, 30, 20, 6, 3, seed=6)

    def spread(t, step):
        wide = torch.zeros(t.shape[0], t.shape[1] * step + 3, dtype=t.dtype, device=t.device)
        view = wide[:, 1:1 + t.shape[1]] if step == 1 else wide[:, 1:1 + t.shape[1] * step:step]
        view.copy_(t)
        return view
    from mamba2_recall import sampling
    want = sampling.adjust(logits, **kw)
    for step in (1, 2):
        views = dict(kw, prompt=spread(kw["prompt"], step), tokens=spread(kw["tokens"], step),
                     bias=tuple(spread(t, step) for t in kw["bias"]), allowed=spread(kw["allowed"], step))
        assert torch.equal(_bits(sampling.adjust(spread(logits, step), **views)), _bits(want))
    expanded = dict(prompt=kw["prompt"][:1].expand(4, -1), tokens=kw["tokens"][:1].expand(4, -1))
    _check(logits, repetition=1.2, frequency=0.1, **expanded)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_extreme_logits(device, dtype):
    top = torch.finfo(dtype).max
    row = [0.0, -0.0, INF, -INF, float("nan"), top, -top, torch.finfo(dtype).tiny, -torch.finfo(dtype).tiny / 4, 1.0]
    logits = torch.tensor([row] * 3, device=device).to(dtype)
    ids = torch.arange(10, device=device).expand(3, -1)
    mask = torch.tensor([[-1], [0], [0b0000010110]], dtype=torch.int32, device=device)
    _check(logits, tokens=ids, repetition=torch.tensor([2.0, 1.0, 0.5], device=device), presence=0.25)
    got = _check(logits, tokens=ids, repetition=1.5, allowed=mask)
    assert bool((got[1] == -INF).all())                       # a NaN that is masked, too
    assert bool(torch.isnan(got[0, 4])) and got[2, 4] != got[2, 4]


def test_sample_after_a_mask_that_leaves_nothing(device):
    from mamba2_recall import sampling
    logits, _ = _case(device, torch.float32, 2, 3000, 0, 0, 0, 0, seed=8)
    words = torch.zeros(2, 94, dtype=torch.int32, device=device)
    words[1, 17] = 1 << 9
    ids, logprobs = sampling.sample(sampling.adjust(logits, allowed=words), torch.full((2,), 0.5, device=device))
    assert ids.tolist() == [-1, 17 * 32 + 9] and logprobs.tolist() == [-INF, 0.0]


def test_other_stream_and_graph(device):
    """Captured with the ids growing in place, replayed between eager work."""
    from mamba2_recall import sampling
    logits, kw = _case(device, torch.float16, 3, 5000, 40, 25, 6, 3, seed=9)
    static = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    src = logits.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = sampling.adjust(src, **static)
    stream.synchronize()
    assert torch.equal(_bits(side), _bits(sampling.adjust(logits, **kw)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampling.adjust(src, **static)
    for step in range(4):
        static["lengths"].fill_(3 + step)
        src.copy_(logits * (step + 1))
        want = sampling.adjust(src, **static)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(_bits(out), _bits(want))


def test_refusals(device):
    from mamba2_recall import sampling
    logits, kw = _case(device, torch.float32, 2, 64, 4, 4, 2, 2, seed=10)
    for change in (dict(out=logits.half()), dict(out=logits[:1]), dict(out=logits.t().contiguous().t()),
                   dict(prompt=kw["prompt"].cpu()), dict(allowed=kw["allowed"].cpu())):
        with pytest.raises(ValueError):
            sampling.adjust(logits, **change)
    buffer = torch.zeros(3, 64, device=device)
    with pytest.raises(ValueError, match="apart"):
        sampling.adjust(buffer[:2], out=buffer[1:])
    with pytest.raises(ValueError, match="apart"):
        sampling.adjust(buffer.flatten()[:128].view(2, 64), out=buffer.flatten()[8:136].view(2, 64))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,vocab,prompt,tokens,wide", [
    (2, 30011, 9000, 40, True), (2, 9001, 0, 8192, False),      # long lists, few rows
    (130, 333, 8150, 60, True), (64, 17001, 8192, 5, False),    # long lists, many rows
    (300, 1000, 30, 20, True), (1, 5000, 4100, 0, True)])       # many rows; a list of some length
def test_launch_shapes(device, dtype, batch, vocab, prompt, tokens, wide):
    logits, kw = _case(device, dtype, batch, vocab, prompt, tokens, 6, 5, seed=batch + vocab, wide=wide)
    _check(logits, **kw)


def test_offsets_past_32_bits(device):
    """More than 2^31 logits: the last rows are those of a small call."""
    from mamba2_recall import sampling
    gen = torch.Generator(device=device).manual_seed(11)
    logits = torch.empty(8500, 256000, dtype=torch.float16, device=device).normal_(generator=gen)
    tokens = torch.randint(0, 256000, (8500, 9), generator=gen, device=device)
    masks = torch.full((1, 8000), -1, dtype=torch.int32, device=device)
    masks[0, 7999] = 0
    kw = dict(presence=0.5, frequency=0.25, repetition=1.1)
    rows = torch.zeros(8500, dtype=torch.int32, device=device)
    last = sampling.adjust(logits[-4:], tokens=tokens[-4:], allowed=masks, allowed_rows=rows[-4:], **kw)
    got = sampling.adjust(logits, tokens=tokens, allowed=masks, allowed_rows=rows, **kw)
    assert torch.equal(got[-4:], last) and bool((got[-1, -32:] == -INF).all())
    del got
    sampling.adjust(logits, tokens=tokens, allowed=masks, allowed_rows=rows, out=logits, **kw)
    assert torch.equal(logits[-4:], last)
