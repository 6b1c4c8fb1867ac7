"""Token sampling with temperature, top-k, top-p and min-p from given uniform
numbers, one a row, and what comes before it: penalties for repeated tokens,
biases and grammar masks on the logits.  The reference decodes greedily
(scripts/infer_fp4_ridge_resurface_v1.py:102-109); runs the gfx950 HIP kernels
of libm2r_hip.so (m2r_adjust_logits, m2r_sample)."""
from __future__ import annotations

import torch

from . import _native

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _filter(value, name, dtype, like, low, high):
    """(tensor or None, scalar) of one filter: a number for every row, or a
    tensor with a value for each."""
    if isinstance(value, torch.Tensor):
        if value.dtype is not dtype or value.shape != (like.shape[0],) or value.device != like.device:
            raise ValueError(f"{name} must be a number or {str(dtype).split('.')[1]}[batch] on the logits' device")
        return value if value.shape[0] < 2 or value.stride(0) == 1 else value.contiguous(), 0
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


def penalties(like, repetition, presence, frequency):
    """The three penalties as (tensor or None, scalar), checked for as many rows
    as `like` has, on its device."""
    return (_filter(repetition, "repetition", torch.float32, like, 1e-30, 1e30),
            _filter(presence, "presence", torch.float32, like, -1e30, 1e30),
            _filter(frequency, "frequency", torch.float32, like, -1e30, 1e30))


# An eager call on small tensors is bound by the host: the checks below ask a
# tensor for its type, shape and device number once each.
def _list(ids, lengths, name, batch, device):
    """A list of ids a row as the C entry takes it: (ids, is int64, row stride, ids a row, lengths)."""
    if ids is None:
        if lengths is not None:
            raise ValueError(f"{name}: lengths without ids")
        return None, 0, 0, 0, None
    if (not isinstance(ids, torch.Tensor) or ids.dtype is not torch.int64 and ids.dtype is not torch.int32
            or ids.ndim != 2 or ids.shape[0] != batch or ids.get_device() != device):
        raise ValueError(f"{name} must be int64 or int32 [batch,ids] on the logits' device")
    if lengths is not None:
        if (not isinstance(lengths, torch.Tensor) or lengths.dtype is not torch.int32 or lengths.shape != (batch,)
                or lengths.get_device() != device):
            raise ValueError(f"The lengths of {name} must be int32[batch] on the logits' device")
        if batch > 1 and lengths.stride(0) != 1:
            lengths = lengths.contiguous()
    stride, unit = ids.stride()
    count = ids.shape[1]
    if count > 1 and unit != 1:
        ids, stride = ids.contiguous(), count
    return ids, ids.dtype is torch.int64, stride, count, lengths


def biases(like, bias):
    """(ids, values), int32 and FP32 [batch,n], of a bias for as many rows as
    `like` has, on its device; (None, None) for no bias."""
    if bias is None:
        return None, None
    if not isinstance(bias, (tuple, list)) or len(bias) != 2 or not all(isinstance(t, torch.Tensor) for t in bias):
        raise ValueError("bias must be a pair of tensors, ids and values")
    ids, values = bias
    batch, shape = like.shape[0], ids.shape
    if (ids.dtype is not torch.int32 or values.dtype is not torch.float32 or shape != values.shape
            or len(shape) not in (1, 2) or len(shape) == 2 and shape[0] != batch
            or not like.get_device() == ids.get_device() == values.get_device()):
        raise ValueError("bias must be int32 ids and FP32 values, both [n] or [batch,n], on the logits' device")
    if len(shape) == 1:
        ids, values = ids.expand(batch, -1), values.expand(batch, -1)
    if shape[-1] > 1:
        ids = ids if ids.stride(1) == 1 else ids.contiguous()
        values = values if values.stride(1) == 1 else values.contiguous()
    return ids, values


def masks(like, vocab, allowed, allowed_rows):
    """(masks int32[masks,words], the row's mask int32[batch] or None), checked
    for as many rows as `like` has, on its device.  `vocab` None: not known
    yet, any number of words passes."""
    if allowed is None:
        if allowed_rows is not None:
            raise ValueError("allowed_rows without allowed")
        return None, None
    words, batch = "words" if vocab is None else (vocab + 31) // 32, like.shape[0]
    if (not isinstance(allowed, torch.Tensor) or allowed.dtype is not torch.int32 or allowed.ndim not in (1, 2)
            or 0 in allowed.shape or vocab is not None and allowed.shape[-1] != words
            or allowed.get_device() != like.get_device()):
        raise ValueError(f"allowed must be int32 [{words}] or [masks,{words}], a bit a token, on the logits' device")
    if allowed.ndim == 1:
        if allowed_rows is not None:
            raise ValueError("allowed_rows needs a list of masks")
        allowed = allowed.expand(batch, -1)
    elif allowed_rows is None:
        if allowed.shape[0] != batch:
            raise ValueError("A mask for each row, or allowed_rows, required")
    elif (not isinstance(allowed_rows, torch.Tensor) or allowed_rows.dtype is not torch.int32
          or allowed_rows.shape != (batch,) or allowed_rows.get_device() != like.get_device()):
        raise ValueError("allowed_rows must be int32[batch] on the logits' device")
    elif batch > 1 and allowed_rows.stride(0) != 1:
        allowed_rows = allowed_rows.contiguous()
    if allowed.shape[1] > 1 and allowed.stride(1) != 1:
        allowed = allowed.contiguous()
    return allowed, allowed_rows


def _span(t):
    """The bytes from a tensor's first element to its last one's end."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def adjust(logits, *, prompt=None, prompt_lengths=None, tokens=None, lengths=None, repetition=1.0, presence=0.0,
           frequency=0.0, bias=None, allowed=None, allowed_rows=None, out=None):
    """Logits with each request's penalties, biases and grammar mask: a new
    tensor of their type and shape, or `out` (`logits` itself, or memory apart
    from them: no rows of one between rows of the other).

    logits[B,V] in FP16, BF16 or FP32 (unit column stride).  `prompt` and
    `tokens` (int64 or int32 [B,n], unit column stride) are the ids that a
    request came with and those generated since; prompt_lengths and lengths
    int32[B] say how many of a row count (default: all; values are clamped to
    0..n); ids outside the vocabulary count for nothing.  Applied in this
    order, in FP32, to a token that is c times among `tokens`:

        repetition   l / r where l > 0, else l * r   if in prompt or tokens
        presence p, frequency f   l - (f c + p)      if c > 0
        bias         l + value: (ids int32, values FP32), both [n] or [B,n]; an
                     id outside the vocabulary is unused, of an id that is named
                     twice the later value counts
        allowed      -inf where bit (token % 32) of word token // 32 is 0:
                     int32 [V/32, rounded up] for all rows, or [masks, words],
                     row b's by allowed_rows[b] (int32[B]; outside the masks
                     for none), by default mask b

    repetition (above 0), presence and frequency are numbers, or FP32[B].  A
    logit that nothing touches keeps its bits, and the others are rounded once
    to their type.  Forward only."""
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError("logits must be CUDA FP16, BF16 or FP32 [batch,vocabulary]")
    batch, vocab = logits.shape
    if vocab < 1:
        raise ValueError("A vocabulary of at least one token required")
    (r, r_all), (pr, pr_all), (f, f_all) = penalties(logits, repetition, presence, frequency)
    device = logits.get_device()
    prompt, p64, ps, pn, prompt_lengths = _list(prompt, prompt_lengths, "prompt", batch, device)
    tokens, t64, ts, tn, lengths = _list(tokens, lengths, "tokens", batch, device)
    ids, values = biases(logits, bias)
    allowed, allowed_rows = masks(logits, vocab, allowed, allowed_rows)
    source = logits
    if vocab > 1 and logits.stride(1) != 1 or batch > 1 and logits.stride(0) < vocab:
        source = logits.contiguous()
    if out is None:
        out = torch.empty_like(source, memory_format=torch.contiguous_format)
    elif out is not logits or source is not logits:
        if (not isinstance(out, torch.Tensor) or out.dtype != logits.dtype or out.shape != logits.shape
                or out.device != logits.device or vocab > 1 and out.stride(1) != 1
                or batch > 1 and out.stride(0) < vocab):
            raise ValueError("out must have the logits' type and shape, and rows of unit stride that do not overlap")
        (o0, o1), (l0, l1) = (_span(out), _span(source)) if batch else ((0, 0), (0, 0))
        if o0 < l1 and l0 < o1 and (o0 != l0 or out.stride() != source.stride()):
            raise ValueError("out must be logits itself or memory apart from it")
    if batch == 0:
        return out
    p = _native.ptr
    n = 0 if ids is None else ids.shape[1]
    with _native.device_of(logits):
        _native.call("m2r_adjust_logits", p(source), _DTYPES[logits.dtype], source.stride(0) if batch > 1 else vocab,
                     p(out), out.stride(0) if batch > 1 else vocab, p(prompt), p64, ps, pn, p(prompt_lengths), p(tokens),
                     t64, ts, tn, p(lengths), p(r), float(r_all), p(pr), float(pr_all), p(f), float(f_all), p(ids),
                     ids.stride(0) if n else 0, p(values), values.stride(0) if n else 0, n, p(allowed),
                     0 if allowed is None else allowed.stride(0), 0 if allowed is None else allowed.shape[0],
                     p(allowed_rows), batch, vocab, _native.stream_of(logits))
    return out


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
