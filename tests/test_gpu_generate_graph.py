"""A decode step of the full-precision controller with adapters and the draw of
the next token, captured into a graph and replayed between eager work."""
import pytest
import torch

from test_gpu_generate import BATCH, VOCAB, _few, _sets, small  # noqa: F401  (small: a fixture)

pytestmark = pytest.mark.gpu


def test_captured_decode_step(small, device):  # noqa: F811
    from mamba2_recall import sampling
    from mamba2_recall.full_state import FullState
    gen = torch.Generator(device=device).manual_seed(9)
    prompt = torch.randint(0, VOCAB, (BATCH, 12), generator=gen, device=device)
    u = torch.rand(BATCH, 9, generator=gen, device=device)
    t = torch.tensor([0.7, 1.0, 0.0], device=device)
    kw = dict(temperature=t, top_k=40, top_p=0.9)
    with _few(FullState, small) as c, torch.no_grad():
        c.use_adapters(_sets(device), torch.tensor([2, -1, 0], dtype=torch.int32, device=device))

        def decode(step):
            hidden = c.backbone(prompt, reset=True)
            token, rows = sampling.sample(small.lm_head(hidden[:, -1]), u[:, 0], **kw)[0], []
            for k in range(1, 9):
                token = step(token, u[:, k])
                rows.append(token.clone())
            return torch.stack(rows, 1)

        def eager(token, number):
            return sampling.sample(small.lm_head(c.backbone(token[:, None])[:, -1]), number.contiguous(), **kw)[0]
        want = decode(eager)
        layers = c._cache
        saved = [(e.conv.clone(), e.state.clone()) for e in layers]
        static_token = torch.zeros(BATCH, dtype=torch.long, device=device)
        static_number = torch.zeros(BATCH, device=device)
        eager(static_token, static_number)       # every kernel and library handle is there before the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = eager(static_token, static_number)
        # the captured request goes back to its prompt, in place
        fresh = _few(FullState, small)
        c.close()
        with fresh:
            fresh.use_adapters(_sets(device), torch.tensor([2, -1, 0], dtype=torch.int32, device=device))
            hidden = fresh.backbone(prompt, reset=True)
            first = sampling.sample(small.lm_head(hidden[:, -1]), u[:, 0], **kw)[0]
            for e, f in zip(layers, fresh._cache):
                e.conv.copy_(f.conv)
                e.state.copy_(f.state)
        static_token.copy_(first)
        for k in range(1, 9):
            static_number.copy_(u[:, k])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[:, k - 1]), f"step {k}"
            static_token.copy_(out)
        assert all(torch.equal(e.state, s) for e, (_, s) in zip(layers, saved))
