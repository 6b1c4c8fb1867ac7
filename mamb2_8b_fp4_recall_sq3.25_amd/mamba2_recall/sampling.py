"""Token sampling with temperature, top-k, top-p and min-p from given uniform
numbers, one a row.  The reference decodes greedily
(scripts/infer_fp4_ridge_resurface_v1.py:102-109); runs the gfx950 HIP kernels
of libm2r_hip.so (m2r_sample)."""
from __future__ import annotations

import torch

from . import _native

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _filter(value, name, dtype, like, low, high):
    """(tensor or None, scalar) of one filter: a number for every row, or a
    tensor with a value for each."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or tuple(value.shape) != (like.shape[0],) or value.device != like.device:
            raise ValueError(f"{name} must be a number or {str(dtype).split('.')[1]}[batch] on the logits' device")
        return value.contiguous(), 0
    if isinstance(value, bool) or not isinstance(value, (int, float) if dtype == torch.float32 else int) \
            or not low <= value <= high:
        raise ValueError(f"{name} must lie in [{low}, {high}]")
    return None, value


def filters(like, temperature, top_k, top_p, min_p):
    """The four filters as (tensor or None, scalar), checked for as many rows as
    `like` has, on its device."""
    return (_filter(temperature, "temperature", torch.float32, like, 0.0, 1e30),
            _filter(top_k, "top_k", torch.int32, like, 0, 2 ** 31 - 1),
            _filter(top_p, "top_p", torch.float32, like, 0.0, 1.0),
            _filter(min_p, "min_p", torch.float32, like, 0.0, 1.0))


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draw one token a row: (ids int64[B], logprobs float32[B]).

    logits[B,V] in FP16, BF16 or FP32 (unit column stride); uniforms FP32[B]
    in [0, 1).  Filters are numbers, or tensors with a value for each row
    (FP32; top_k int32), applied in this order: temperature (0: the likeliest
    token, the lowest index of equal ones; a tensor's may be infinite: all
    tokens above -inf alike), top_k (0: off; equal logits in
    the order of their indices), top_p of what top_k left (the shortest
    prefix of the sorted row that holds it, at least one token), min_p
    relative to the likeliest token.  The token is found by the inverse of
    the distribution function in the order of the indices; its log
    probability is that of the filtered distribution.

    Weights are whole multiples of 2^-31 of the likeliest token's, so sums
    are exact and a result does not depend on the launch; tokens below that
    are never drawn.  A NaN logit counts as -inf; a row with nothing above
    -inf gives the id -1 and the log probability -inf."""
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError("logits must be CUDA FP16, BF16 or FP32 [batch,vocabulary]")
    batch, vocab = logits.shape
    if vocab < 1:
        raise ValueError("A vocabulary of at least one token required")
    if (not isinstance(uniforms, torch.Tensor) or uniforms.dtype != torch.float32 or tuple(uniforms.shape) != (batch,)
            or uniforms.device != logits.device):
        raise ValueError("uniforms must be FP32[batch] on the logits' device")
    (t, t_all), (k, k_all), (tp, tp_all), (mp, mp_all) = filters(logits, temperature, top_k, top_p, min_p)
    ids = logits.new_empty(batch, dtype=torch.int64)
    logprobs = torch.empty_like(uniforms, memory_format=torch.contiguous_format)
    if batch == 0:
        return ids, logprobs
    if vocab > 1 and logits.stride(1) != 1 or batch > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    uniforms = uniforms.contiguous()
    per_row = t is not None or k is not None or tp is not None
    ws_bytes = int(_native.lib().m2r_sample_call_workspace(batch, vocab, per_row, float(t_all), k_all, float(tp_all)))
    ws = logits.new_empty(ws_bytes, dtype=torch.uint8)
    p = _native.ptr
    with _native.device_of(logits):
        _native.call("m2r_sample", p(logits), _DTYPES[logits.dtype], logits.stride(0) if batch > 1 else vocab,
                     p(uniforms), p(t), float(t_all), p(k), k_all, p(tp), float(tp_all), p(mp), float(mp_all), p(ids),
                     p(logprobs), batch, vocab, p(ws), ws_bytes, _native.stream_of(logits))
    return ids, logprobs
