"""The full-precision controller, adapters of many requests and sampling
together, on a model of two layers of the real geometry, against a
restatement of the whole model in 64 bits.

Tolerance (derived): every value between two modules is rounded to binary16
(about twelve roundings a layer, 2^-11 relative at most, about 2^-12.8 in the
mean square each, independent): 2 layers give sqrt(24) 2^-12.8 = 7e-4; taken
as 4e-3 for the sums' own spread."""
import math

import pytest
import torch

import mamba2_model

pytestmark = pytest.mark.gpu

LAYERS, VOCAB, BATCH = 2, 4000, 3


@pytest.fixture(scope="module")
def small(device):
    with torch.device("meta"):
        model = mamba2_model.Mamba2LM(layers=LAYERS, vocab=VOCAB)
    model = model.to_empty(device=device).half().requires_grad_(False).eval()
    gen = torch.Generator(device=device).manual_seed(3)
    for name, p in model.named_parameters():
        if name.endswith("A_log"):
            p.copy_(torch.log(torch.rand(p.shape, generator=gen, device=device) * 15 + 1))
        elif name.endswith("dt_bias"):
            p.copy_(torch.log(torch.expm1(torch.rand(p.shape, generator=gen, device=device) * 0.09 + 0.01)))
        elif "norm" in name:
            p.fill_(1.0)
        elif name.endswith("conv1d.bias"):
            p.zero_()
        elif name.endswith(".D"):
            p.copy_(torch.randn(p.shape, generator=gen, device=device))
        else:
            p.normal_(0.0, 1.0 / math.sqrt(p.shape[-1]), generator=gen)
    return model


def _few(cls, model, *args):
    params = list(model.parameters())
    few = type("Few" + cls.__name__, (cls,), dict(LAYERS=LAYERS, TABLE_SHAPE=(LAYERS, 8, 128), PARAMETER_TENSORS=len(params),
                                                  PARAMETER_COUNT=sum(p.numel() for p in params)))
    return few(model, *args)


def _sets(device, rank=16, count=4):
    from mamba2_recall import adapters
    gen = torch.Generator(device=device).manual_seed(5)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)
    out = []
    for _ in range(LAYERS):
        out.append({name: adapters.AdapterSet((normal(count, rank, k) / k ** 0.5).half(),
                                              (normal(count, n, rank) / rank ** 0.5).half(),
                                              torch.full((count,), 0.5, device=device))
                    for name, k, n in (("in_proj", 4096, 18560), ("out_proj", 8192, 4096))})
    return out


def _project64(mx, name, sets, ids, v):
    out = v @ getattr(mx, name).weight.double().T
    if sets is not None:
        s = sets[name]
        for b, a in enumerate(ids.tolist()):
            if 0 <= a < s.count:
                out[b] += s.scale[a].double() * ((v[b] @ s.down[a].double().T) @ s.up[a].double().T)
    return out


def _backbone64(model, prompt, sets, ids):
    def rms(v, w, eps):
        return v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    hidden, residual = model.backbone.embedding.weight[prompt].double(), None
    batch, tokens = prompt.shape
    for i, layer in enumerate(model.backbone.layers):
        mx = layer.mixer
        residual = hidden if residual is None else hidden + residual
        u = rms(residual, layer.norm.weight, layer.norm.eps)
        zx = _project64(mx, "in_proj", None if sets is None else sets[i], ids, u)
        z, xbc, dt = torch.split(zx, (8192, 10240, 128), dim=-1)
        w = mx.conv1d.weight.double()[:, 0]
        padded = torch.cat((torch.zeros_like(xbc[:, :1]).expand(-1, 3, -1), xbc), 1)
        conv = sum(padded[:, k:k + tokens] * w[:, k] for k in range(4)) + mx.conv1d.bias.double()
        x, bm, cm = torch.split(conv * torch.sigmoid(conv), (8192, 1024, 1024), dim=-1)
        x = x.reshape(batch, tokens, 128, 64)
        bm, cm = (t.reshape(batch, tokens, 8, 128).repeat_interleave(16, 2) for t in (bm, cm))
        v = dt + mx.dt_bias.double()
        step = torch.logaddexp(v, torch.zeros_like(v))
        decay = torch.exp(-torch.exp(mx.A_log.double()) * step)
        s = torch.zeros(batch, 128, 64, 128, dtype=torch.float64, device=x.device)
        ys = []
        for t in range(tokens):
            s = s * decay[:, t, :, None, None] + (step[:, t, :, None] * x[:, t])[..., None] * bm[:, t, :, None]
            ys.append((s * cm[:, t, :, None]).sum(-1) + mx.D.double()[:, None] * x[:, t])
        y = torch.stack(ys, 1).flatten(-2) * (z * torch.sigmoid(z))
        y = y.unflatten(-1, (8, -1))
        y = (y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + mx.norm.eps)).flatten(-2) * mx.norm.weight.double()
        hidden = _project64(mx, "out_proj", None if sets is None else sets[i], ids, y)
    return rms(hidden + residual, model.backbone.norm_f.weight, model.backbone.norm_f.eps)


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("tokens", [1, 30, 100])
@pytest.mark.parametrize("adapted", [False, True])
def test_model_against_64_bits(small, device, tokens, adapted):
    """A prompt in one call, and the same prompt with its last token as a step."""
    from mamba2_recall.full_state import FullState
    gen = torch.Generator(device=device).manual_seed(tokens)
    prompt = torch.randint(0, VOCAB, (BATCH, tokens), generator=gen, device=device)
    sets = _sets(device) if adapted else None
    ids = torch.tensor([2, -1, 0], dtype=torch.int32, device=device)
    want = _backbone64(small, prompt, sets, ids)
    with _few(FullState, small) as c:
        c.use_adapters(sets, ids)
        assert _rel(c.backbone(prompt, reset=True), want) < 4e-3
        assert c.assert_finite_cache() and c.cache_breakdown()["tokens_per_layer"] == [tokens] * LAYERS
        if tokens > 1:
            c.backbone(prompt[:, :-1], reset=True)
            assert _rel(c.backbone(prompt[:, -1:]), want[:, -1:]) < 4e-3


@pytest.mark.parametrize("packed", [False, True])
def test_rows_without_an_adapter_keep_their_bits(small, device, packed):
    """Any controller takes adapters; a request without one is untouched."""
    from mamba2_recall.state_quant import StateQuant
    from test_gpu_controllers import _g16_packets
    prompt = torch.randint(0, VOCAB, (2, 9), generator=torch.Generator(device=device).manual_seed(1), device=device)
    with _few(StateQuant, small, "s16") as c:
        if packed:
            c.use_packed_projections(_g16_packets(small, device, 7))
        def run():
            return torch.cat((c.backbone(prompt[:, :8], reset=True), c.backbone(prompt[:, 8:])), 1)
        plain = run()
        c.use_adapters(_sets(device), torch.tensor([-1, 3], dtype=torch.int32, device=device))
        got = run()
        assert torch.equal(got[0], plain[0]) and not torch.equal(got[1], plain[1])
        c.use_adapters(None)
        assert torch.equal(run(), plain)


def test_generate(small, device):
    """Greedy rows follow the argmax; the same numbers give the same tokens;
    each row's tokens come from its filtered distribution."""
    from mamba2_recall.full_state import FullState
    from mamba2_recall.generate import generate
    gen = torch.Generator(device=device).manual_seed(2)
    prompt = torch.randint(0, VOCAB, (BATCH, 20), generator=gen, device=device)
    u = torch.rand(BATCH, 6, generator=gen, device=device)
    t = torch.tensor([0.0, 0.8, 1.0], device=device)
    k = torch.tensor([0, 5, 0], dtype=torch.int32, device=device)
    with _few(FullState, small) as c:
        c.use_adapters(_sets(device), torch.tensor([1, 1, -1], dtype=torch.int32, device=device))
        ids, logprobs = generate(c, small.lm_head, prompt, u, temperature=t, top_k=k)
        again = generate(c, small.lm_head, prompt, u, temperature=t, top_k=k)
        assert torch.equal(ids, again[0]) and torch.equal(logprobs, again[1])
        assert bool(((ids >= 0) & (ids < VOCAB)).all()) and bool((logprobs <= 0).all())
        assert bool((logprobs[0] == 0).all())
        hidden = c.backbone(prompt, reset=True)
        for s in range(6):
            logits = small.lm_head(hidden[:, -1])
            assert int(logits[0].argmax()) == int(ids[0, s])
            assert int(ids[1, s]) in logits[1].float().topk(5).indices.tolist()
            p = torch.log_softmax(logits[2].double(), 0)[ids[2, s]]
            assert abs(float(p) - float(logprobs[2, s])) < 1e-4
            hidden = c.backbone(ids[:, s:s + 1])
        with pytest.raises(ValueError):
            generate(c, small.lm_head, prompt, u[:2])
        with pytest.raises(ValueError):
            generate(c, small.lm_head, prompt, u[:, :0])


def test_adapter_refusals(small, device):
    from mamba2_recall import adapters
    from mamba2_recall.full_state import FullState
    sets, ids = _sets(device), torch.zeros(BATCH, dtype=torch.int32, device=device)
    c = _few(FullState, small)
    wrong = adapters.AdapterSet(sets[0]["out_proj"].down, sets[0]["out_proj"].up)
    for s, i in ((sets[:1], ids), (sets, None), (sets, ids.long()), (sets, ids.cpu()), ([dict(in_proj=wrong), None], ids),
                 ([dict(x_proj=wrong), None], ids), ([dict(out_proj=wrong.down), None], ids)):
        with pytest.raises(ValueError):
            c.use_adapters(s, i)
    with c:
        c.use_adapters(sets, ids)
        with pytest.raises(ValueError):
            c.backbone(torch.zeros(2, 4, dtype=torch.long, device=device), reset=True)
