"""A queue of prompts of different lengths through the full-precision
controller, projections and head in 8-bit integers, penalties, biases and masks
on the logits: together, as generate() runs them, and each step by itself, on a
model of two layers of the real geometry."""
import textwrap

import pytest
import torch

from test_gpu_generate import BATCH, LAYERS, VOCAB, _few, _rel, _sets, small  # noqa: F401  (small: a fixture)
from test_gpu_generate import _backbone64

pytestmark = pytest.mark.gpu

NAMES = ("in_proj", "out_proj")


def _weights(model):
    from mamba2_recall.int8 import Int8Weight
    return [{name: Int8Weight.quantize(getattr(layer.mixer, name).weight) for name in NAMES}
            for layer in model.backbone.layers]


def _prompts(device, tokens, seed=1):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(0, VOCAB, (BATCH, tokens), generator=gen, device=device), gen


def _int32(device, *values):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("counts", [(100, 1, 37), (3, 100, 64), (100, 100, 100)])
def test_rows_of_different_lengths(small, device, counts):  # noqa: F811
    """Every row against the model in 64 bits over its own tokens (the bound of
    test_gpu_generate), in one call and with its last token as a step; what
    stands behind a row's tokens changes nothing."""
    from mamba2_recall.full_state import FullState
    prompt, gen = _prompts(device, 100)
    lengths = _int32(device, *counts)
    other = prompt.clone()
    for i, n in enumerate(counts):
        other[i, n:] = torch.randint(0, VOCAB, (100 - n,), generator=gen, device=device)
    nxt = torch.randint(0, VOCAB, (BATCH, 1), generator=gen, device=device)
    with _few(FullState, small) as c:
        hidden = c.backbone(prompt, reset=True, lengths=lengths)
        states = [(e.conv.clone(), e.state.clone()) for e in c._cache]
        again = c.backbone(other, reset=True, lengths=lengths)
        step = c.backbone(nxt)
        assert c.assert_finite_cache()
        for i, n in enumerate(counts):
            want = _backbone64(small, torch.cat((prompt[i:i + 1, :n], nxt[i:i + 1]), 1), None, None)
            assert _rel(hidden[i:i + 1, :n], want[:, :n]) < 4e-3
            assert _rel(step[i:i + 1], want[:, n:]) < 4e-3
            assert torch.equal(hidden[i, :n], again[i, :n])
        c.backbone(other, reset=True, lengths=lengths)
        for e, (conv, state) in zip(c._cache, states):
            assert torch.equal(e.conv, conv) and torch.equal(e.state, state)


def test_rows_continue_and_rest(small, device):  # noqa: F811
    """A second call of several tokens, and of one, with lengths: a row of none
    keeps its caches."""
    from mamba2_recall.full_state import FullState
    prompt, _ = _prompts(device, 40, seed=2)
    with _few(FullState, small) as c:
        c.backbone(prompt[:, :20], reset=True, lengths=_int32(device, 20, 5, 11))
        before = [(e.conv.clone(), e.state.clone()) for e in c._cache]
        c.backbone(prompt[:, 20:30], lengths=_int32(device, 0, 10, 3))
        c.backbone(prompt[:, 30:31], lengths=_int32(device, 0, 1, 0))
        rest = [(e.conv[0].clone(), e.state[0].clone()) for e in c._cache]
        got = c.backbone(prompt[:, 31:32])
        for (conv, state), (conv0, state0) in zip(rest, before):
            assert torch.equal(conv, conv0[0]) and torch.equal(state, state0[0])
        rows = (torch.cat((prompt[0, :20], prompt[0, 31:32])),
                torch.cat((prompt[1, :5], prompt[1, 20:30], prompt[1, 30:32])),
                torch.cat((prompt[2, :11], prompt[2, 20:23], prompt[2, 31:32])))
        for i, row in enumerate(rows):
            want = _backbone64(small, row[None], None, None)
            assert _rel(got[i:i + 1], want[:, -1:]) < 4e-3


def test_int8_projections(small, device):  # noqa: F811
    """The projections' modules replaced by 8-bit products: each equals
    int8.linear of its own input, and the whole stays within the codes' own
    distance of the model whose weights are the decoded codes."""
    from mamba2_recall import int8
    from mamba2_recall.full_state import FullState
    weights = _weights(small)
    prompt, _ = _prompts(device, 70, seed=3)
    seen = []
    real = int8.linear

    def spy(x, weight, dtype=None):
        y = real(x, weight, dtype)
        seen.append((tuple(x.shape), weight))
        return y
    with _few(FullState, small) as c:
        plain = c.backbone(prompt, reset=True)
        c.use_int8_projections(weights)
        int8.linear = spy
        try:
            got = c.backbone(prompt, reset=True)
            step = c.backbone(prompt[:, :1])
        finally:
            int8.linear = real
        order = [w for entry in weights for w in (entry["in_proj"], entry["out_proj"])]
        assert [s[1] for s in seen] == order * 2
        assert [s[0] for s in seen[:2]] == [(BATCH, 70, 4096), (BATCH, 70, 8192)]
        assert [s[0] for s in seen[2 * LAYERS:2 * LAYERS + 2]] == [(BATCH, 4096), (BATCH, 8192)]
        # A code is off by up to half a step of 1/127 of its row's or channel's largest value, uniformly: 0.29 steps in
        # the mean square.  The largest of thousands of normal values is about four deviations, so a factor is off by
        # 0.29 * 4 / 127 = 0.9% of its deviation, a product of two by 1.3%; four products and what the norms and gates
        # make of them: taken as 8%.
        assert _rel(got, plain.double()) < 0.08 and not torch.equal(got, plain)
        # off again, and for one layer and one projection only
        c.use_int8_projections(None)
        assert torch.equal(c.backbone(prompt, reset=True), plain)
        c.use_int8_projections([None, dict(out_proj=weights[1]["out_proj"])])
        some = c.backbone(prompt, reset=True)
        assert not torch.equal(some, plain) and _rel(some, plain.double()) < 0.08
        assert torch.equal(c.backbone(prompt[:, :1]).isfinite(), torch.ones_like(step, dtype=torch.bool))


def test_packed_steps_go_before_int8(small, device):  # noqa: F811
    """Packed FP4 projections keep the one-token calls that they take."""
    from mamba2_recall import fp4, int8
    from mamba2_recall.full_state import FullState
    from test_gpu_controllers import _g16_packets
    prompt, _ = _prompts(device, 5, seed=4)
    with _few(FullState, small) as c:
        packets = _g16_packets(small, device, 7)
        c.use_packed_projections(packets)
        c.use_int8_projections(_weights(small))
        calls = []
        real8, real4 = int8.linear, fp4.gemv_g16
        int8.linear = lambda *a: calls.append("int8") or real8(*a)
        fp4.gemv_g16 = lambda *a: calls.append("fp4") or real4(*a)
        try:
            c.backbone(prompt[:2], reset=True)
            c.backbone(prompt[:2, :1])
            c.backbone(prompt, reset=True)
            c.backbone(prompt[:, :1])        # three rows: not for the packed product
        finally:
            int8.linear, fp4.gemv_g16 = real8, real4
    n = 2 * LAYERS
    assert calls == ["int8"] * n + ["fp4"] * n + ["int8"] * n * 2


def test_generate_adjusts_each_step(small, device):  # noqa: F811
    """generate()'s tokens are those of the calls one after the other, with the
    prompts' own tokens and those drawn so far in the penalties, and a grammar
    that follows what was drawn."""
    from mamba2_recall import int8, sampling
    from mamba2_recall.full_state import FullState
    from mamba2_recall.generate import generate
    prompt, gen = _prompts(device, 30, seed=5)
    lengths = _int32(device, 30, 4, 17)
    u = torch.rand(BATCH, 6, generator=gen, device=device)
    head = int8.Int8Weight.quantize(small.lm_head.weight)
    words = VOCAB // 32
    ids = torch.randint(0, VOCAB, (BATCH, 9), generator=gen, device=device, dtype=torch.int32)
    values = torch.randn(BATCH, 9, generator=gen, device=device)
    repetition = torch.tensor([1.0, 1.3, 1.1], device=device)

    def logits_of(rows):
        return head(rows, torch.float32)

    def grammar(drawn):
        """No token that is a neighbour of the last one in its word; anything first."""
        if drawn.shape[1] == 0:
            return None
        masks = torch.full((BATCH, words), -1, dtype=torch.int32, device=device)
        return masks.scatter_(1, drawn[:, -1:] // 32, 0)
    kw = dict(temperature=0.9, top_k=50)
    extra = dict(repetition=repetition, presence=0.4, frequency=0.3, bias=(ids, values))
    with _few(FullState, small) as c:
        c.use_int8_projections(_weights(small))
        c.use_adapters(_sets(device), _int32(device, 1, -1, 2))
        got, logprobs = generate(c, logits_of, prompt, u, lengths=lengths, allowed=grammar, **kw, **extra)
        hidden = c.backbone(prompt, reset=True, lengths=lengths)
        last = torch.stack([hidden[i, n - 1] for i, n in enumerate(lengths.tolist())])
        drawn = torch.zeros(BATCH, 0, dtype=torch.int64, device=device)
        for s in range(6):
            logits = sampling.adjust(logits_of(last), prompt=prompt, prompt_lengths=lengths, tokens=drawn,
                                     allowed=grammar(drawn), **extra)
            token, logprob = sampling.sample(logits, u[:, s].contiguous(), **kw)
            assert torch.equal(got[:, s], token) and torch.equal(logprobs[:, s], logprob)
            if s:
                assert not bool((token // 32 == drawn[:, -1] // 32).any())
            drawn = torch.cat((drawn, token[:, None]), 1)
            last = c.backbone(token[:, None])[:, -1]


def test_generate_without_settings_is_unchanged(small, device):  # noqa: F811
    from mamba2_recall.full_state import FullState
    from mamba2_recall.generate import generate
    prompt, gen = _prompts(device, 12, seed=6)
    u = torch.rand(BATCH, 5, generator=gen, device=device)
    with _few(FullState, small) as c:
        plain = generate(c, small.lm_head, prompt, u, top_k=20)
        same = generate(c, small.lm_head, prompt, u, top_k=20, repetition=1, presence=0, frequency=0.0, allowed=lambda d: None)
        assert all(torch.equal(a, b) for a, b in zip(plain, same))
        bans = torch.zeros(VOCAB // 32, dtype=torch.int32, device=device)
        none = generate(c, small.lm_head, prompt, u, allowed=bans)
        assert bool((none[0] == -1).all()) and bool(torch.isinf(none[1]).all())


def test_refusals(small, device):  # noqa: F811
    from mamba2_recall.full_state import FullState
    from mamba2_recall.generate import generate
    from mamba2_recall.int8 import Int8Weight
    from mamba2_recall.state_quant import StateQuant
    prompt, gen = _prompts(device, 6, seed=7)
    u = torch.rand(BATCH, 2, generator=gen, device=device)
    lengths = _int32(device, 6, 2, 3)
    weights = _weights(small)
    with _few(StateQuant, small, "s16") as c:
        with pytest.raises(ValueError, match="one length"):
            c.backbone(prompt, reset=True, lengths=lengths)
        assert c.use_int8_projections(weights).backbone(prompt, reset=True).isfinite().all()
    with _few(FullState, small) as c:
        c.backbone(prompt, reset=True)
        for bad in (lengths.long(), lengths[:2], lengths.cpu(), [6, 2, 3]):
            with pytest.raises(ValueError, match="lengths"):
                c.backbone(prompt, lengths=bad)
            with pytest.raises(ValueError, match="lengths"):
                generate(c, small.lm_head, prompt, u, lengths=bad)
        assert c.cache_breakdown()["tokens_per_layer"] == [6] * LAYERS       # the request is as it was
        wrong = Int8Weight.quantize(small.lm_head.weight)
        for bad in (weights[:1], [dict(in_proj=wrong), None], [dict(x_proj=wrong), None],
                    [dict(in_proj=small.lm_head.weight), None]):
            with pytest.raises(ValueError):
                c.use_int8_projections(bad)
        handle = small.backbone.layers[0].mixer.act.register_forward_hook(lambda *a: None)
        try:
            with pytest.raises(ValueError, match="plain"):
                c.backbone(prompt, reset=True, lengths=lengths)
        finally:
            handle.remove()


def test_example_runs(small, device, monkeypatch):  # noqa: F811
    """The example in the 8-bit projections' documentation, as it is written."""
    from mamba2_recall import full_state, generate, int8
    text = int8.__doc__
    code = textwrap.dedent("\n".join(line for line in text[text.index("    weights = "):].splitlines()
                                     if line.startswith("    ") or not line.strip()))
    assert "generate.generate(" in code and "use_int8_projections" in code
    cls = full_state.FullState
    monkeypatch.setattr(full_state, "FullState", lambda model: _few(cls, model))
    prompt, gen = _prompts(device, 9, seed=8)
    names = dict(int8=int8, full_state=full_state, generate=generate, torch=torch, model=small, prompt=prompt,
                 uniforms=torch.rand(BATCH, 4, generator=gen, device=device), lengths=_int32(device, 3, 9, 1),
                 bias_ids=_int32(device, 5, 6), bias_values=torch.tensor([2.0, -3.0], device=device),
                 masks=torch.full((VOCAB // 32,), -2, dtype=torch.int32, device=device))
    exec(compile(code, "example", "exec"), names)
    new = names["new"]
    assert new.shape == names["logprobs"].shape == (BATCH, 4)
    assert bool(((new >= 0) & (new < VOCAB) & (new % 32 != 0)).all())


@pytest.mark.parametrize("padding", [-1, VOCAB + 7, 1 << 40])
def test_padding_of_any_value(small, device, padding):  # noqa: F811
    """Prompts filled up with ids outside the vocabulary give what those filled up with tokens give."""
    from mamba2_recall import generate
    from mamba2_recall.full_state import FullState
    prompt, gen = _prompts(device, 30, seed=8)
    lengths = _int32(device, 30, 4, 17)
    padded = prompt.clone()
    for i, n in enumerate(lengths.tolist()):
        padded[i, n:] = padding
    uniforms = torch.rand(BATCH, 3, generator=gen, device=device)
    head = torch.nn.functional.linear
    weight = torch.randn(VOCAB, small.backbone.layers[0].mixer.in_proj.weight.shape[1], generator=gen, device=device).half()
    with _few(FullState, small) as c:
        def run(ids):
            return generate.generate(c, lambda rows: head(rows, weight).float(), ids, uniforms, lengths=lengths,
                                     repetition=1.2, presence=0.1)
        (ids, logprobs), (same, same_logprobs) = run(prompt), run(padded)
    assert torch.equal(ids, same) and torch.equal(logprobs, same_logprobs)
