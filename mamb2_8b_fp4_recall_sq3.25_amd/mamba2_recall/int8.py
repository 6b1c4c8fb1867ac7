"""Projections in 8-bit integers, a scale for each token and each output channel.

A server keeps a projection's weights in an Int8Weight, half the bytes of
FP16; `linear` gives each token's row a scale of its own, from its largest
value, and multiplies the whole numbers:

    s[m] = max|x[m]| / 127,  q[m] = round(127 x[m] / max|x[m]|)
    y[m] = s[m] * scale * (q[m] @ codes.T)

The reference keeps decoded FP16 weights for all its projections
(mamba2_recall/fp4_checkpoint.py:345-405); this is for prompts and batches,
where fp4.gemv_g16 ends.  A queue of prompts of different lengths, projections
and head in 8-bit integers, with penalties, biases and a grammar for each:

    weights = [{name: int8.Int8Weight.quantize(getattr(layer.mixer, name).weight) for name in ("in_proj", "out_proj")}
               for layer in model.backbone.layers]
    head = int8.Int8Weight.quantize(model.lm_head.weight)
    with full_state.FullState(model) as controller:
        controller.use_int8_projections(weights)
        new, logprobs = generate.generate(controller, lambda rows: head(rows, torch.float32), prompt, uniforms,
                                          lengths=lengths, temperature=0.8, top_p=0.95, repetition=1.1, frequency=0.2,
                                          bias=(bias_ids, bias_values), allowed=lambda drawn: masks)

Runs the gfx950 HIP kernels of libm2r_hip.so (m2r_int8_quantize,
m2r_int8_linear)."""
from __future__ import annotations

import torch

from . import _native

MAX_INPUTS = 131072          # sums of that many products fit 32 bits
MAX_CHANNELS = 1 << 24       # of a product
MAX_QUANTIZED = MAX_CHANNELS - 128   # channels whose codes one launch forms: 256 threads each, fewer than 2^32

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


# The kernels read weights in tiles of 16 channels by 64 inputs.  Of 32 channels
# the first tile has the first four
# of every eight; N is filled up to a multiple of 32, K to one of 128.
def _groups(n, k):
    return (n + 31) // 32, (k + 127) // 128 * 2


def _geometry(shape, channels):
    n, k = shape
    if min(n, k) < 1 or k > MAX_INPUTS or n > channels:
        raise ValueError(f"Positive geometry, at most {MAX_INPUTS} inputs and {channels} channels required")
    return n, k


class Int8Weight:
    """The weights of one projection: `codes` int8[N,K] and `scale` FP32[N] (N
    at most 2^24, K at most 131,072), the value of a weight being its code times
    its channel's scale.  Kept in the order in which the kernels read them; call
    it, or `linear`, with rows of K."""

    def __init__(self, codes, scale):
        if not isinstance(codes, torch.Tensor) or codes.dtype != torch.int8 or codes.ndim != 2 or not codes.is_cuda:
            raise ValueError("codes must be CUDA int8[N,K]")
        n, k = _geometry(codes.shape, MAX_CHANNELS)
        if (not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or tuple(scale.shape) != (n,)
                or scale.device != codes.device):
            raise ValueError("scale must be FP32[N] on the device of codes")
        groups, steps = _groups(n, k)
        filled = torch.nn.functional.pad(codes, (0, 64 * steps - k, 0, 32 * groups - n))
        self.features = k, n
        self.tiles = filled.view(groups, 4, 2, 4, steps, 4, 16).permute(0, 2, 4, 5, 1, 3, 6).contiguous()
        self.scale = scale.detach().clone(memory_format=torch.contiguous_format)

    @classmethod
    def quantize(cls, weight):
        """FP16 or BF16 weights [N,K] (N at most 16,777,088), each channel by
        its largest value.  A channel with a value that is not finite has the
        scale NaN."""
        if (not isinstance(weight, torch.Tensor) or weight.dtype not in (torch.float16, torch.bfloat16)
                or weight.ndim != 2 or not weight.is_cuda):
            raise ValueError("weight must be CUDA FP16 or BF16 [N,K]")
        n, k = _geometry(weight.shape, MAX_QUANTIZED)
        self = cls.__new__(cls)
        self.features = k, n
        weight, stride = _rows(weight.detach(), k)
        groups, steps = _groups(n, k)
        self.tiles = torch.zeros((groups, 2, steps, 4, 4, 4, 16), dtype=torch.int8, device=weight.device)
        self.scale = torch.empty(n, dtype=torch.float32, device=weight.device)
        with _native.device_of(weight):
            _native.call("m2r_int8_quantize", _native.ptr(weight), _TYPES[weight.dtype], stride, _native.ptr(self.tiles),
                         _native.ptr(self.scale), n, k, _native.stream_of(weight))
        return self

    @property
    def codes(self):
        """int8[N,K]."""
        k, n = self.features
        groups, steps = _groups(n, k)
        return self.tiles.permute(0, 4, 1, 5, 2, 3, 6).reshape(32 * groups, 64 * steps)[:n, :k]

    def decode(self, dtype=torch.float16):
        """The weights' values [N,K], rounded once."""
        return (self.codes.float() * self.scale[:, None]).to(dtype)

    def __call__(self, x, dtype=None):
        return linear(x, self, dtype)


def _rows(t, features):
    """`t` [rows, features] with unit column stride, and its row stride."""
    stride, column = t.stride()
    if column != 1 and features > 1 or t.shape[0] > 1 and stride < features:
        t, stride = t.contiguous(), features
    return t, stride if t.shape[0] > 1 else features


def linear(x, weight, dtype=None):
    """x[..., K] in FP16 or BF16 times an Int8Weight: a new tensor [..., N] of
    x's type, or of `dtype` (FP16, BF16 or FP32).

    The sum of a row's products is exact, its product with the two scales is
    formed in FP32 and rounded once, so a row's result depends on the row
    alone.  A row with a value that is not finite gives NaN; two scales whose
    product overflows FP32 give infinities, and NaN for a sum of 0.  Forward
    only."""
    if not isinstance(weight, Int8Weight):
        raise ValueError("weight must be an Int8Weight")
    k, n = weight.features
    if (not isinstance(x, torch.Tensor) or x.dtype not in (torch.float16, torch.bfloat16) or not x.is_cuda or x.ndim < 1
            or x.shape[-1] != k or x.device != weight.tiles.device):
        raise ValueError(f"x must be FP16 or BF16 [..., {k}] on the weights' device")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _TYPES:
        raise ValueError("dtype must be FP16, BF16 or FP32")
    rows, stride = _rows(x if x.ndim == 2 else x.reshape(-1, k), k)
    m = rows.shape[0]
    y = torch.empty((*x.shape[:-1], n), dtype=dtype, device=x.device)
    if m == 0:
        return y
    at, p = rows.data_ptr(), _native.ptr
    ws_bytes = _native.lib().m2r_int8_linear_workspace(at, stride, m, n, k)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    with _native.device_of(x):
        _native.call("m2r_int8_linear", at, _TYPES[x.dtype], stride, p(weight.tiles), p(weight.scale), p(y),
                     _TYPES[dtype], n, m, n, k, p(ws), ws_bytes, _native.stream_of(x))
    return y
