"""The example of many requests in the generation module's documentation runs as
it is written, on a model of two layers of the real geometry."""
import textwrap

import pytest
import torch

from test_gpu_generate import BATCH, VOCAB, _few, small  # noqa: F401  (small: a fixture)

pytestmark = pytest.mark.gpu


def test_example_runs(small, device, monkeypatch):  # noqa: F811
    from mamba2_recall import adapters, full_state, generate
    lines = generate.__doc__.splitlines()
    code = textwrap.dedent("\n".join(line for line in lines if line.startswith("    ") or not line.strip()))
    assert "generate.generate(" in code
    cls = full_state.FullState
    monkeypatch.setattr(full_state, "FullState", lambda model: _few(cls, model))
    gen = torch.Generator(device=device).manual_seed(1)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)
    names = dict(
        adapters=adapters, full_state=full_state, generate=generate, model=small, lm_head=small.lm_head,
        weights=[((normal(2, 8, 4096) / 64).half(), (normal(2, 18560, 8) / 4).half(), torch.ones(2, device=device))
                 for _ in range(2)],
        ids=torch.tensor([1, -1, 0], dtype=torch.int32, device=device),
        prompt=torch.randint(0, VOCAB, (BATCH, 7), generator=gen, device=device),
        uniforms=torch.rand(BATCH, 4, generator=gen, device=device))
    exec(compile(code, "example", "exec"), names)
    assert names["new"].shape == names["logprobs"].shape == (BATCH, 4)
    assert bool(((names["new"] >= 0) & (names["new"] < VOCAB)).all())


def test_controller_must_be_installed(small, device):  # noqa: F811
    from mamba2_recall.full_state import FullState
    from mamba2_recall.generate import generate
    with pytest.raises(RuntimeError, match="not installed"):
        generate(_few(FullState, small), small.lm_head, torch.zeros(1, 2, dtype=torch.long, device=device),
                 torch.zeros(1, 1, device=device))
