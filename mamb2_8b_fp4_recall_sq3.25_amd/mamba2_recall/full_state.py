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


def _check(x, dt, A, B, C, D, dt_bias, state, lengths, slots):
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
    if B.ndim != 4:
        raise ValueError("B must have four axes")
    groups = B.shape[2]
    if groups < 1 or heads % groups:
        raise ValueError("heads must be divisible by B/C groups")
    shapes = ((dt, (batch, length, heads)), (A, (heads,)), (B, (batch, length, groups, N)),
              (C, (batch, length, groups, N)), (D, (heads,)), (dt_bias, (heads,)))
    for t, shape in shapes:
        if tuple(t.shape) != shape or t.device != x.device:
            raise ValueError("Input device/geometry mismatch")
    if A.dtype != torch.float32 or any(t.dtype != torch.float16 for t in (dt, B, C)):
        raise ValueError("A must be FP32; dt/B/C must be FP16")
    if any(t.dtype not in (torch.float16, torch.float32) for t in (D, dt_bias)):
        raise ValueError("D and dt_bias must be FP16 or FP32")
    for name, t in (("lengths", lengths), ("slots", slots)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (batch,)
                              or t.device != x.device):
            raise ValueError(f"{name} must be int32[batch] on the device of x")
    return batch, length, heads, dim, groups


def _token_rows(t):
    """`t` [batch, tokens, ...] with dense trailing dimensions and its two
    leading strides; any view whose tokens are dense rows is read in place."""
    inner = 1
    for size, stride in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if size > 1 and stride != inner:
            t = t.contiguous()
            break
        inner *= size
    return t, t.stride(0), t.stride(1)


@torch.no_grad()
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
    later tokens non-finite, and no earlier ones."""
    geo = _check(x, dt, A, B, C, D, dt_bias, state, lengths, slots)
    (x, *xs), (dt, *ds), (B, *bs), (C, *cs) = map(_token_rows, (x, dt, B, C))
    A, D, dt_bias = A.contiguous(), D.contiguous(), dt_bias.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    slots = None if slots is None else slots.contiguous()
    y = torch.empty(x.shape, dtype=torch.float16, device=x.device)
    ws_bytes = int(_native.lib().m2r_full_scan_workspace(*geo))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    p = _native.ptr
    with _native.device_of(x):
        _native.call("m2r_full_scan", p(x), *xs, p(dt), *ds, p(A), p(B), *bs, p(C), *cs, p(D),
                     int(D.dtype == torch.float32), p(dt_bias), int(dt_bias.dtype == torch.float32), p(state),
                     state.shape[0], p(slots), p(lengths), p(y), *geo, p(ws), ws_bytes, _native.stream_of(x))
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
