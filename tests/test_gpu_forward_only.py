"""The queue's operators take tensors that require gradients and return results
that do not, as their documentation says."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_results_carry_no_graph(device):
    from mamba2_recall import full_state, int8, sampling
    for f in (int8.linear, sampling.adjust, full_state.convolve):
        assert "Forward only" in " ".join(f.__doc__.split())
    x = torch.randn(3, 32, device=device).half().requires_grad_()
    weight = int8.Int8Weight.quantize(torch.randn(8, 32, device=device).half().requires_grad_())
    assert not int8.linear(x, weight).requires_grad and not weight.tiles.requires_grad and not weight.scale.requires_grad
    given = int8.Int8Weight(weight.codes, torch.ones(8, device=device, requires_grad=True))
    assert not int8.linear(x, given).requires_grad and not given.scale.requires_grad
    logits = torch.randn(2, 40, device=device, requires_grad=True)
    bias = (torch.zeros(1, dtype=torch.int32, device=device), torch.ones(1, device=device, requires_grad=True))
    assert not sampling.adjust(logits, bias=bias).requires_grad
    value = torch.randn(2, 5, 32, device=device).half().requires_grad_()
    taps = torch.randn(32, 4, device=device).half().requires_grad_()
    parts = full_state.convolve(value, taps, None, full_state.allocate_windows(2, 32, device), (16, 8, 8))
    assert not any(p.requires_grad for p in parts)
