"""Adapters: each kernel instance and each way of dealing rows, by rank and by
number of rows, against the formula in 64 bits (test_gpu_adapters' tolerance)."""
import pytest
import torch

from test_gpu_adapters import _add, _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [65, 96, 100, 128])
@pytest.mark.parametrize("rows", [1, 17, 65, 300])
def test_ranks_of_four_steps(device, rows, rank):
    """Ranks of 65 to 128."""
    c = _case(device, rows, 520, 200, 3, rank, seed=rank + rows)
    _check(c, _add(c))


@pytest.mark.parametrize("rank", [8, 32, 33, 64, 80, 128, 200])
@pytest.mark.parametrize("rows", [513, 1500, 4096])
def test_prompts(device, rows, rank):
    """513 to 4,096 rows, mixed and as runs of one request's rows; ranks on both
    sides of 64, where two tiles stop sharing the second launch's weights."""
    c = _case(device, rows, 600, 330, 4, rank, seed=rank)
    _check(c, _add(c))
    c["ids"] = (torch.arange(rows, device=device) // 217 % 6 - 1).to(torch.int32)
    _check(c, _add(c))


@pytest.mark.parametrize("rank", [72, 130, 256])
def test_many_rows_of_high_rank(device, rank):
    """More than 4,096 rows with more than 64 ranks: the first launch's loop
    over the ranks goes round more than once."""
    c = _case(device, 4112, 136, 72, 3, rank, seed=rank)
    _check(c, _add(c))
