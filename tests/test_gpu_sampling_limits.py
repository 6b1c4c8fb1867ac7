"""Sampling at the ends of its filters' ranges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 1001, 30003])
@pytest.mark.parametrize("kw", [{}, dict(top_k=3), dict(top_p=0.7), dict(top_k=400, top_p=0.9, min_p=0.5)])
def test_endless_temperature(device, dtype, vocab, kw):
    """An infinite temperature (and the largest finite one) makes all tokens
    that are not masked equally likely, and no others: weights are exact, so
    the token is known."""
    from mamba2_recall import sampling
    gen = torch.Generator(device=device).manual_seed(vocab)
    logits = torch.randn(6, vocab, generator=gen, device=device).to(dtype)
    logits[:, 1::4] = -math.inf
    logits[:, 2::4] = math.nan
    u = torch.tensor([0.0, 0.2, 0.5, 0.9, 1.0 - 2.0 ** -24, 0.7], device=device)
    t = torch.tensor([math.inf, math.inf, 3.0e38, math.inf, math.inf, 1.0e30], device=device)
    ids, lp = sampling.sample(logits, u, temperature=t, **kw)
    for b in range(6):
        l = logits[b].float().cpu()
        order = torch.sort(torch.nan_to_num(l, nan=-math.inf), descending=True, stable=True).indices
        n = int(torch.isfinite(l).sum())
        n = min(n, kw.get("top_k", 0) or n)
        if "top_p" in kw:   # the shortest prefix of n equal weights that holds it
            n = math.ceil(math.ceil(float(torch.tensor(kw["top_p"])) * n * 2 ** 31) / 2 ** 31)
        kept = torch.sort(order[:n]).values
        assert int(ids[b]) == int(kept[min(int(math.floor(float(u[b]) * n * 2 ** 31)) // 2 ** 31, n - 1)]), b
        assert abs(float(lp[b]) + math.log(n)) < 1e-5
