"""Every way in which a product in 8-bit integers is cut, in every output type
and with channels that are and are not whole eights, against whole numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [
    # few rows: codes in the product's launch, and beside it; 32 channels a workgroup, and 64
    (1, 8200, 256), (2, 8200, 256), (3, 8200, 256), (4, 8200, 250), (20, 8200, 256), (40, 8200, 320), (64, 8200, 200),
    (1, 65600, 128), (4, 65600, 128), (10, 65600, 128), (30, 65600, 130), (60, 65600, 128),
    # few channels: inputs split among workgroups
    (9, 4096, 4096), (25, 2048, 8192), (50, 72, 4096), (100, 1000, 4096), (128, 4096, 1024),
    # blocks of a quarter's size, and split inputs
    (130, 40, 8192), (200, 512, 4096), (400, 1000, 2100), (300, 2048, 256),
    # large blocks; the last round's in halves; in quarters; a round and a rest
    (4096, 2816, 128), (2560, 2560, 192), (2048, 2048, 256), (2000, 18560, 128), (5000, 4090, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("m,n,k", CASES)
def test_instance(device, m, n, k, odd, dtype):
    from mamba2_recall.int8 import Int8Weight, linear
    n -= odd
    gen = torch.Generator(device=device).manual_seed(m + n + k)
    codes = torch.randint(-127, 128, (n, k), generator=gen, device=device, dtype=torch.int8)
    scale = (torch.rand(n, generator=gen, device=device) + 0.5) / 127 / k ** 0.5
    x = torch.randn(m, k, generator=gen, device=device).to(torch.float16 if odd else torch.bfloat16)
    got = linear(x, Int8Weight(codes, scale), dtype)
    xd = x.double()
    top = xd.abs().amax(1, keepdim=True)
    q = torch.round(127.0 * xd / top).float()
    want = torch.zeros(m, n, dtype=torch.float64, device=device)
    for i in range(0, k, 1024):      # sums of 1,024 products are exact in binary32
        want += (q[:, i:i + 1024] @ codes[:, i:i + 1024].float().T).double()
    want *= top / 127 * scale.double()
    # half a step of the type, five binary32 roundings, half a step of binary16's subnormals
    bound = want.abs() * (torch.finfo(dtype).eps / 2 + 5 * 2.0 ** -24) + 2.0 ** -25
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())
