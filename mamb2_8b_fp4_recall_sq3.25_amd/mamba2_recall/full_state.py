"""Selective-state scan with a full-precision (FP32) carry, and its controller.

The unquantized control that every packed carry is judged against: linear
attention with a decay for each head, as the Mamba-2 mixer runs it
(reference: the native recurrence that mamba2_recall/state_codec.py:65-102
rounds to FP16 after every token).  The carries of many requests live in one
pool, FP32[slots,H,P,128]; a call names the slot and the token count of each
batch row, so prompts of different lengths and idle rows share a launch.
convolve is the mixer's convolution before it, over a pool of windows in the
same manner.  They run the gfx950 HIP kernels of libm2r_hip.so (m2r_full_scan,
m2r_conv_pool).
"""
from __future__ import annotations

import torch
from torch import nn

from . import _native
from .state_quant import _MixerController, _plain

N = 128


def allocate_state(slots, heads, dim, dstate, device):
    """A zeroed pool of carries, FP32 [slots, heads, dim, 128]."""
    if dstate != N or min(slots, heads, dim) <= 0:
        raise ValueError("Require dstate=128 and positive geometry")
    return torch.zeros((slots, heads, dim, N), dtype=torch.float32, device=device)


def _refuse(x, dt, A, B, C, D, dt_bias, state, lengths, slots):
    """The reason why a call is not taken."""
    if not isinstance(x, torch.Tensor) or x.ndim != 4 or x.dtype != torch.float16 or not x.is_cuda:
        raise ValueError("x must be CUDA FP16[batch,tokens,heads,dim]")
    batch, length, heads, dim = x.shape
    if min(batch, length, heads, dim) < 1:
        raise ValueError("Positive geometry required")
    if (not isinstance(state, torch.Tensor) or state.dtype != torch.float32 or state.ndim != 4
            or tuple(state.shape[1:]) != (heads, dim, N) or state.shape[0] < 1 or state.device != x.device
            or not state.is_contiguous()):
        raise ValueError("state must be contiguous FP32[slots,heads,dim,128] on the device of x")
    if slots is None and state.shape[0] < batch:
        raise ValueError("A carry for every batch row, or slots, required")
    if not isinstance(B, torch.Tensor) or B.ndim != 4:
        raise ValueError("B must have four axes")
    groups = B.shape[2]
    if groups < 1 or heads % groups:
        raise ValueError("heads must be divisible by B/C groups")
    shapes = ((dt, (batch, length, heads)), (A, (heads,)), (B, (batch, length, groups, N)),
              (C, (batch, length, groups, N)), (D, (heads,)), (dt_bias, (heads,)))
    for t, shape in shapes:
        if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape or t.device != x.device:
            raise ValueError("Input device/geometry mismatch")
    if A.dtype != torch.float32 or any(t.dtype != torch.float16 for t in (dt, B, C)):
        raise ValueError("A must be FP32; dt/B/C must be FP16")
    if any(t.dtype not in (torch.float16, torch.float32) for t in (D, dt_bias)):
        raise ValueError("D and dt_bias must be FP16 or FP32")
    for name, t in (("lengths", lengths), ("slots", slots)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (batch,)
                              or t.device != x.device):
            raise ValueError(f"{name} must be int32[batch] on the device of x")


def _taken(x, dt, A, B, C, D, dt_bias, state, lengths, slots):
    """The same conditions at once, for the call that meets them: a step of a
    few microseconds is bound by the host."""
    try:
        batch, length, heads, dim = xs = x.shape
        groups = B.shape[2]
        bc, h, dev, f16, f32, i32 = (batch, length, groups, N), (heads,), x.device, torch.float16, torch.float32, torch.int32
        return (x.dtype is f16 and x.is_cuda and 0 not in xs and state.dtype is f32 and state.is_contiguous()
                and state.shape[1:] == (heads, dim, N) and state.shape[0] >= (1 if slots is not None else batch)
                and groups > 0 and heads % groups == 0 and dt.shape == xs[:3] and B.shape == bc and C.shape == bc
                and A.shape == h and D.shape == h and dt_bias.shape == h and A.dtype is f32
                and dt.dtype is f16 and B.dtype is f16 and C.dtype is f16
                and (D.dtype is f16 or D.dtype is f32) and (dt_bias.dtype is f16 or dt_bias.dtype is f32)
                and state.device == dt.device == A.device == B.device == C.device == D.device == dt_bias.device == dev
                and (lengths is None or lengths.dtype is i32 and lengths.shape == (batch,) and lengths.device == dev)
                and (slots is None or slots.dtype is i32 and slots.shape == (batch,) and slots.device == dev))
    except (AttributeError, ValueError, IndexError):
        return False


def _token_rows(t):
    """`t` [batch, tokens, ...] and its strides of batch rows and tokens; any
    view whose tokens are dense rows is read in place."""
    s, n = t.stride(), t.shape
    dense = s[2] == 1 or n[2] == 1 if len(n) == 3 else (s[3] == 1 or n[3] == 1) and (s[2] == n[3] or n[2] == 1)
    if not dense:
        t = t.contiguous()
        s = t.stride()
    return t, s[0], s[1]


def scan(x, dt, A, B, C, D, dt_bias, state, *, lengths=None, slots=None):
    """Advance carries over the tokens of x; return (FP16 readouts, None).

    x[B,L,H,P], dt[B,L,H], B/C[B,L,G,128] in FP16 (views with dense tokens are
    read in place); A[H] FP32, D[H] and dt_bias[H] FP16/FP32.  `state` is the
    FP32[S,H,P,128] pool, changed in place.  `slots` int32[B] names each batch
    row's carry: negative, or not below S, for an idle row, and no slot twice
    (default: row b uses carry b).  `lengths` int32[B] is each row's token
    count (default: L; values are clamped to 0..L).  Readouts past a row's
    length, and an idle row's, are zero; the carry stands after the row's last
    token.  A non-finite input makes the affected readouts of its own and
    later tokens non-finite, and no earlier ones.  Forward only."""
    if not _taken(x, dt, A, B, C, D, dt_bias, state, lengths, slots):
        _refuse(x, dt, A, B, C, D, dt_bias, state, lengths, slots)
    batch, length, heads, dim = x.shape
    groups = B.shape[2]
    x, xb, xl = _token_rows(x)
    dt, db, dl = _token_rows(dt)
    B, bb, bl = _token_rows(B)
    C, cb, cl = _token_rows(C)
    A, D, dt_bias = A.contiguous(), D.contiguous(), dt_bias.contiguous()
    lengths = lengths.contiguous() if lengths is not None else None
    slots = slots.contiguous() if slots is not None else None
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    ws, ws_bytes = None, 0
    if length > 1:
        ws_bytes = _native.lib().m2r_full_scan_workspace(batch, length, heads, dim, groups)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    p = _native.ptr
    with _native.device_of(x):
        _native.call("m2r_full_scan", x.data_ptr(), xb, xl, dt.data_ptr(), db, dl, A.data_ptr(), B.data_ptr(), bb, bl,
                     C.data_ptr(), cb, cl, D.data_ptr(), D.dtype is torch.float32, dt_bias.data_ptr(),
                     dt_bias.dtype is torch.float32, state.data_ptr(), state.shape[0], p(slots), p(lengths),
                     y.data_ptr(), batch, length, heads, dim, groups, p(ws), ws_bytes, _native.stream_of(x))
    return y, None


def allocate_windows(slots, channels, device):
    """A zeroed pool of convolution windows, FP16 [slots, channels, 4] with the
    channels next to each other in memory."""
    if min(slots, channels) <= 0:
        raise ValueError("Positive geometry required")
    return torch.zeros((slots, 4, channels), dtype=torch.float16, device=device).permute(0, 2, 1)


def convolve(value, weight, bias, window, sizes, *, lengths=None, slots=None, silu=True):
    """The mixer's short causal convolution with SiLU over a pool of windows,
    as scan takes its carries: the channels of `sizes` as three contiguous FP16
    tensors [B,L,n].

    value FP16[B,L,C] (a view with dense tokens is read in place), weight
    FP16[C,4], bias FP16[C] or None; `window` FP16[S,C,4] (allocate_windows) is
    the pool, changed in place: a row's last four inputs, of which the last
    three precede its tokens; zeros for a new request.  `slots` and `lengths`
    are scan's: outputs past a row's length, and an idle row's, are zero, and an
    idle or empty row leaves its window alone.  The sum and the SiLU are formed
    in FP32 and rounded once.  Forward only."""
    if not isinstance(value, torch.Tensor) or value.dtype != torch.float16 or value.ndim != 3 or not value.is_cuda:
        raise ValueError("value must be CUDA FP16[batch,tokens,channels]")
    batch, tokens, channels = value.shape
    if batch < 1 or tokens < 1 or channels < 1:
        raise ValueError("Positive geometry required")
    if not isinstance(sizes, (tuple, list)) or len(sizes) != 3 \
            or not all(isinstance(n, int) and n > 0 for n in sizes) or sum(sizes) != channels:
        raise ValueError("sizes must be three positive channel counts that add up to value's")
    # (a call of one token is bound by the host: each tensor is asked once)
    f16, device, rows = torch.float16, value.get_device(), (batch,)
    if not isinstance(weight, torch.Tensor) or weight.dtype is not f16 or weight.shape != (channels, 4) \
            or weight.get_device() != device:
        raise ValueError(f"weight must be FP16[{channels}, 4] on the device of value")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.dtype is not f16 or bias.shape != (channels,)
                             or bias.get_device() != device):
        raise ValueError(f"bias must be FP16[{channels}] on the device of value")
    if (not isinstance(window, torch.Tensor) or window.dtype is not f16 or window.ndim != 3
            or window.shape[1:] != (channels, 4) or window.shape[0] < 1 or window.get_device() != device):
        raise ValueError("window must be FP16[slots,channels,4] on the device of value")
    pool = window.shape[0]
    ws_s, ws_c, ws_t = window.stride()
    if channels > 1 and ws_c != 1 or ws_t < channels or pool > 1 and ws_s < 3 * ws_t + channels:
        raise ValueError("window must have its channels next to each other and none twice (allocate_windows)")
    if slots is None and pool < batch:
        raise ValueError("A window for every batch row, or slots, required")
    for name, t in (("lengths", lengths), ("slots", slots)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.shape != rows
                              or t.get_device() != device):
            raise ValueError(f"{name} must be int32[batch] on the device of value")
    if channels > 1 and value.stride(2) != 1:
        value = value.contiguous()
    if not weight.is_contiguous() or weight.data_ptr() % 8:
        weight = weight.clone(memory_format=torch.contiguous_format)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    lengths = lengths.contiguous() if lengths is not None else None
    slots = slots.contiguous() if slots is not None else None
    x, b, c = (value.new_empty((batch, tokens, n)) for n in sizes)
    vs_b, vs_l, _ = value.stride()
    p = _native.ptr
    with _native.device_of(value):
        _native.call("m2r_conv_pool", window.data_ptr(), pool, ws_s, ws_t, value.data_ptr(), vs_b, vs_l, weight.data_ptr(),
                     p(bias), p(slots), p(lengths), x.data_ptr(), b.data_ptr(), c.data_ptr(), *sizes, batch, tokens, 4,
                     1 if silu else 0, _native.stream_of(value))
    return [x, b, c]


class FullState(_MixerController):
    """Controller with the full-precision carry: prompts in one scan call a
    layer, of different lengths if backbone() is given them, decode one token
    at a time, no table and no quantization."""

    ragged = True

    def __init__(self, model):
        super().__init__(model, "full", None, False)

    def _validate_permutations(self, values):
        return None

    def _new_state(self, batch_size, index):
        return allocate_state(batch_size, self.HEADS, self.HEADDIM, self.D_STATE, self.device)

    def _scan_layer(self, index, mx, x, dt, aa, bm, cm, entry):
        return scan(x, dt, aa, bm, cm, mx.D, mx.dt_bias, entry.state, lengths=self._lengths)

    def _refuse_ragged(self):
        if not all(_plain(mx.conv1d, nn.Conv1d) and _plain(mx.act, nn.SiLU) for mx in self._mixers):
            raise ValueError("Rows of different lengths need a plain nn.Conv1d and nn.SiLU, without hooks")

    def _conv_prefill(self, mx, xbc, layer):
        if self._lengths is None:
            return super()._conv_prefill(mx, xbc, layer)
        return convolve(xbc, mx.conv1d.weight[:, 0, :], mx.conv1d.bias, layer.conv, self._conv_sizes,
                        lengths=self._lengths)

    def assert_finite_cache(self):
        """True when every window and carry is finite, else FloatingPointError."""
        for index, entry in enumerate(self._cache):
            if not bool(torch.isfinite(entry.conv).all() & torch.isfinite(entry.state).all()):
                raise FloatingPointError(f"Non-finite cache in layer {index}")
        return True

    def cache_breakdown(self):
        """Bytes the request holds per kind of tensor, and the places of a row
        that each layer was called with: the padding of rows of different
        lengths counts, as the rows' own tokens are known to the device only."""
        layers = self._cache
        conv = sum(c.conv.numel() * c.conv.element_size() for c in layers)
        state = sum(c.state.numel() * c.state.element_size() for c in layers)
        return {"mode": self.mode, "batch_size": self._batch_size, "allocated_layers": len(layers),
                "conv_fp16_bytes": conv, "ssm_total_bytes": state, "total_bytes": conv + state,
                "tokens_per_layer": [c.tokens for c in layers]}
