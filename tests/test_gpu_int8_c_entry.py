"""What the C entries of the 8-bit projections promise beside int8.linear: rows
of y further apart than they are long, with what lies between them left alone,
and weights whose bytes past the last channel hold anything."""
import pytest
import torch

from mamba2_recall import _native, int8

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = {F16: 0, BF16: 1, F32: 2}
SENTINEL = 0x5a

# rows, channels, inputs: codes formed in the product's launch, few rows, few rows split, small blocks, small blocks
# split, large blocks, large blocks with a cut last round
SHAPES = [(1, 96, 256), (3, 104, 512), (20, 200, 300), (64, 8200, 128), (9, 96, 32768), (100, 104, 8192), (300, 2048, 256),
          (200, 104, 16384), (600, 4096, 192), (2560, 2560, 192), (2000, 18560, 128)]


def _case(device, m, n, k):
    gen = torch.Generator(device=device).manual_seed(m + n + k)
    codes = torch.randint(-127, 128, (n, k), generator=gen, device=device, dtype=torch.int8)
    scale = (torch.rand(n, generator=gen, device=device) + 0.5) / 127 / k ** 0.5
    return torch.randn(m, k, generator=gen, device=device).half(), int8.Int8Weight(codes, scale)


def _linear(x, tiles, scale, y, y_stride, n):
    m, k = x.shape
    need = _native.lib().m2r_int8_linear_workspace(x.data_ptr(), k, m, n, k)
    ws = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device=x.device)   # whatever it held before
    _native.call("m2r_int8_linear", x.data_ptr(), TYPES[x.dtype], k, tiles.data_ptr(), scale.data_ptr(), y.data_ptr(),
                 TYPES[y.dtype], y_stride, m, n, k, ws.data_ptr(), need, _native.stream_of(x))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_rows_apart(device, m, n, k, dtype):
    """Stores of 16 bytes (whole eights of channels, an even stride, whole
    words) and of single values; from the first place of the buffer and from
    its second."""
    x, weight = _case(device, m, n, k)
    want = int8.linear(x, weight, dtype)
    behind = 70
    for gap, first, channels in ((0, 0, n), (2, 0, n), (3, 0, n), (6, 1, n), (40, 2, n), (5, 0, n - 3), (2, 0, n - 1)):
        stride = n + gap
        raw = torch.full(((first + m * stride + behind) * want.element_size(),), SENTINEL, dtype=torch.uint8, device=device)
        store = raw.view(dtype)
        _linear(x, weight.tiles, weight.scale, store[first:], stride, channels)
        rows = store[first:first + m * stride].view(m, stride)
        assert torch.equal(rows[:, :channels], want[:, :channels])
        rows[:, :channels] = torch.full((want.element_size(),), SENTINEL, dtype=torch.uint8, device=device).view(dtype)
        assert bool((raw == SENTINEL).all())


@pytest.mark.parametrize("m", [1, 4, 20, 64, 100, 300, 700])
@pytest.mark.parametrize("n", [1, 31, 97, 1003])
def test_bytes_past_the_last_channel(device, m, n):
    gen = torch.Generator(device=device).manual_seed(n)
    w = torch.randn(n, 512, generator=gen, device=device).half()
    x = torch.randn(m, 512, generator=gen, device=device).half()
    weight = int8.Int8Weight.quantize(w)
    want = int8.linear(x, weight, F32)
    for fill in (0x7f, 0x80, 0xff):
        tiles = torch.full((_native.lib().m2r_int8_weight_bytes(n, 512),), fill, dtype=torch.uint8, device=device)
        scale = torch.full((n + 8,), float("nan"), device=device)
        _native.call("m2r_int8_quantize", w.data_ptr(), 0, 512, tiles.data_ptr(), scale.data_ptr(), n, 512,
                     _native.stream_of(w))
        assert torch.equal(scale[:n], weight.scale) and bool(torch.isnan(scale[n:]).all())
        y = torch.empty(m, n, dtype=F32, device=device)
        _linear(x, tiles, scale, y, n, n)
        assert torch.equal(y, want)
