"""Adjusted logits in rows that are apart: what lies between and behind them is
neither read as logits nor written."""
import pytest
import torch

from test_gpu_adjust import _bits, _case

pytestmark = pytest.mark.gpu

SENTINEL = 0x5a


def _rows(raw, dtype, first, batch, stride, vocab):
    return raw.view(dtype)[first:first + batch * stride].view(batch, stride)[:, :vocab]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,vocab,tokens", [(1, 1000, 30), (3, 1001, 30), (5, 4099, 5000), (64, 16390, 40), (16, 16390, 9000),
                                                (130, 333, 9000), (2, 7, 3)])
def test_between_the_rows(device, dtype, batch, vocab, tokens):
    from mamba2_recall import sampling
    logits, kw = _case(device, dtype, batch, vocab, tokens, tokens, 9, 3, seed=batch)
    want = _bits(sampling.adjust(logits, **kw))
    size = logits.element_size()
    for gap, first in ((1, 0), (3, 1), (8, 8), (40, 5)):
        stride = vocab + gap
        raw = torch.full(((first + batch * stride + 64) * size,), SENTINEL, dtype=torch.uint8, device=device)
        fill = raw[:size].clone().view(dtype)
        # into memory of that stride
        out = _rows(raw, dtype, first, batch, stride, vocab)
        assert sampling.adjust(logits, out=out, **kw) is out and torch.equal(_bits(out), want)
        # from it, and in place
        out.copy_(logits)
        assert torch.equal(_bits(sampling.adjust(out, **kw)), want)
        assert sampling.adjust(out, out=out, **kw) is out and torch.equal(_bits(out), want)
        out.copy_(fill.expand(batch, vocab))
        assert bool((raw == SENTINEL).all())
