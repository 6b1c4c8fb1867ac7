"""The 8-bit projections of a controller: which layer's weights meet which
input, bit for bit, and how far the codes of the rows alone move the model."""
import pytest
import torch

from test_gpu_generate import BATCH, LAYERS, VOCAB, _few, _rel, small  # noqa: F401  (small: a fixture)
from test_gpu_generate_queue import NAMES, _int32, _prompts, _weights

pytestmark = pytest.mark.gpu


@pytest.fixture
def projections(small):  # noqa: F811
    """Puts a function of (layer, name, input) in place of every projection's
    computation: the modules run, with what they are given."""
    modules = [(i, name, getattr(layer.mixer, name)) for i, layer in enumerate(small.backbone.layers) for name in NAMES]

    def install(f):
        for i, name, module in modules:
            module.forward = lambda u, i=i, name=name: f(i, name, u)
    yield install
    for _, _, module in modules:
        module.__dict__.pop("forward", None)


def _runs(c, prompt, lengths):
    """Prompts, a continuation of several tokens, single tokens, and rows of
    different lengths."""
    out = [c.backbone(prompt[:, :40], reset=True), c.backbone(prompt[:, 40:47]), c.backbone(prompt[:, 47:48]),
           c.backbone(prompt[:, 48:49])]
    hidden = c.backbone(prompt, reset=True, lengths=lengths)
    out += [hidden[i, :n] for i, n in enumerate(lengths.tolist())]
    return out + [c.backbone(prompt[:, :1])]


def test_each_projection_is_the_product_of_its_own_input_and_weights(small, device, projections):  # noqa: F811
    """The controller's 8-bit products against the modules' places, in which
    the same product is formed from what the module is called with."""
    from mamba2_recall import int8
    from mamba2_recall.full_state import FullState
    weights = _weights(small)
    prompt, _ = _prompts(device, 60, seed=11)
    lengths = _int32(device, 60, 1, 33)
    with _few(FullState, small) as c:
        got = _runs(c.use_int8_projections(weights), prompt, lengths)
        one = _runs(c.use_int8_projections([None, {"out_proj": weights[1]["out_proj"]}]), prompt, lengths)
        c.use_int8_projections(None)
        plain = _runs(c, prompt, lengths)
        projections(lambda i, name, u: int8.linear(u, weights[i][name]))
        assert all(torch.equal(a, b) for a, b in zip(got, _runs(c, prompt, lengths)))
        modules = small.backbone.layers
        projections(lambda i, name, u: int8.linear(u, weights[i][name]) if (i, name) == (1, "out_proj") else
                    torch.nn.functional.linear(u, getattr(modules[i].mixer, name).weight))
        assert all(torch.equal(a, b) for a, b in zip(one, _runs(c, prompt, lengths)))
        # another layer's weights are another result
        projections(lambda i, name, u: int8.linear(u, weights[LAYERS - 1 - i][name]))
        assert not any(torch.equal(a, b) for a, b in zip(got, _runs(c, prompt, lengths)))
    assert not any(torch.equal(a, b) for a, b in zip(got, plain))


def test_distance_from_the_model_of_the_decoded_codes(small, device, projections):  # noqa: F811
    """Against the model whose weights are the decoded codes only the rows'
    codes differ.  A code is off by up to half a step of 1/127 of its row's
    largest value, uniformly: sqrt(1/12) steps in the mean square, which over
    the row's own mean square is the relative error r of a product (sums of many
    independent errors).  Four products, independent; a gated product of four
    projected factors (x, B, C, z) has up to twice its projection's relative
    error, the step's exponential the rest: three times the root of their
    squares' sum, and binary16's own 4e-3 (test_gpu_generate)."""
    from mamba2_recall import int8
    from mamba2_recall.full_state import FullState
    weights = _weights(small)
    decoded = [{name: w.decode(torch.float32) for name, w in entry.items()} for entry in weights]
    prompt, _ = _prompts(device, 60, seed=12)
    squares = []

    def product(i, name, u):
        v = u.float()
        step = v.abs().amax(-1, keepdim=True) / 127
        squares.append(float((step.square() / 12 / v.square().mean(-1, keepdim=True)).mean()))
        return (v @ decoded[i][name].T).half()
    with _few(FullState, small) as c:
        projections(product)
        want = c.backbone(prompt, reset=True)
        assert len(squares) == 2 * LAYERS
        bound = 3 * sum(squares) ** 0.5 + 4e-3
        got = c.use_int8_projections(weights).backbone(prompt, reset=True)
        # the formula's weights rounded to binary16 are the decoded model that a program would load
        projections(lambda i, name, u: torch.nn.functional.linear(u, weights[i][name].decode()))
        loaded = c.use_int8_projections(None).backbone(prompt, reset=True)
    print("distance %.4f, of the decoded weights in FP16 %.4f, bound %.4f" % (_rel(got, want.double()), _rel(loaded, want.double()), bound))
    assert 0 < _rel(got, want.double()) < bound < 0.25
    assert _rel(loaded, want.double()) < 4e-3
