"""Selective-state scan with a full-precision (FP32) carry, and its controller.

The unquantized control that every packed carry is judged against: linear
attention with a decay for each head, as the Mamba-2 mixer runs it
(reference: the native recurrence that mamba2_recall/state_codec.py:65-102
rounds to FP16 after every token).  The carries of many requests live in one
pool, FP32[slots,H,P,128]; a call names the slot and the token count of each
batch row, so prompts of different lengths and idle rows share a launch.
The scan runs the gfx950 HIP kernels of libm2r_hip.so (m2r_full_scan).
"""
from __future__ import annotations

import torch

from . import _native
from .state_quant import _MixerController

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


class FullState(_MixerController):
    """Controller with the full-precision carry: prompts in one scan call a
    layer, decode one token at a time, no table and no quantization."""

    def __init__(self, model):
        super().__init__(model, "full", None, False)

    def _validate_permutations(self, values):
        return None

    def _new_state(self, batch_size, index):
        return allocate_state(batch_size, self.HEADS, self.HEADDIM, self.D_STATE, self.device)

    def _scan_layer(self, index, mx, x, dt, aa, bm, cm, entry):
        return scan(x, dt, aa, bm, cm, mx.D, mx.dt_bias, entry.state)

    def assert_finite_cache(self):
        """True when every window and carry is finite, else FloatingPointError."""
        for index, entry in enumerate(self._cache):
            if not bool(torch.isfinite(entry.conv).all() & torch.isfinite(entry.state).all()):
                raise FloatingPointError(f"Non-finite cache in layer {index}")
        return True

    def cache_breakdown(self):
        """Bytes the request holds per kind of tensor."""
        layers = self._cache
        conv = sum(c.conv.numel() * c.conv.element_size() for c in layers)
        state = sum(c.state.numel() * c.state.element_size() for c in layers)
        return {"mode": self.mode, "batch_size": self._batch_size, "allocated_layers": len(layers),
                "conv_fp16_bytes": conv, "ssm_total_bytes": state, "total_bytes": conv + state,
                "tokens_per_layer": [c.tokens for c in layers]}
