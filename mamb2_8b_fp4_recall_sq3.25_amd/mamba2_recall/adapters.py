"""Low-rank adapters of many requests at once, beside a shared projection.

A server keeps the adapters of one projection in an AdapterSet; `add` gives
every row its own request's update in one call, whatever the mix of adapters:

    out[m] = base[m] + scale[a] * (x[m] @ down[a].T) @ up[a].T,  a = ids[m]

The reference has one adapter for all requests, installed as module hooks
(mamba2_recall/resurface_native.py:363-375).  The products run the gfx950 HIP
kernels of libm2r_hip.so (m2r_adapters_add)."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _native

MAX_RANK = 256


def _aligned(t):
    """`t` from a 16-byte boundary on, which a view may not be."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


class AdapterSet:
    """The adapters of one projection: `down` FP16[n,rank,K], `up`
    FP16[n,N,rank], `scale` FP32[n] (default 1).  Adapters of a lower rank
    are padded with zero rows of `down` and columns of `up`."""

    def __init__(self, down, up, scale=None):
        for t, name in ((down, "down"), (up, "up")):
            if not isinstance(t, torch.Tensor) or t.ndim != 3 or t.dtype != torch.float16 or not t.is_cuda:
                raise ValueError(f"{name} must be CUDA FP16 with three axes")
        n, rank, _ = down.shape
        if min(down.shape) < 1 or min(up.shape) < 1 or rank > MAX_RANK:
            raise ValueError(f"Positive geometry and a rank of at most {MAX_RANK} required")
        if up.shape[0] != n or up.shape[2] != rank or up.device != down.device:
            raise ValueError("down [n,rank,K] and up [n,N,rank] differ in adapters, rank or device")
        if scale is None:
            scale = torch.ones(n, dtype=torch.float32, device=down.device)
        if (not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or tuple(scale.shape) != (n,)
                or scale.device != down.device):
            raise ValueError("scale must be FP32[n] on the adapters' device")
        self.count, self.rank = n, rank
        self.features = down.shape[2], up.shape[1]     # (K, N) of the projection
        # the kernels read ranks and inputs in eights: zeros fill the last
        fill, tail = -rank % 8, -down.shape[2] % 8
        self.down = _aligned(F.pad(down, (0, tail, 0, fill)) if fill or tail else down.contiguous())
        self.up = _aligned(F.pad(up, (0, fill)) if fill else up.contiguous())
        self.scale = scale.contiguous()


def _rows(t, features, what):
    """`t` [..., features] as FP16 rows with unit column stride: (t, rows, row stride)."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or not t.is_cuda or t.ndim < 1 \
            or t.shape[-1] != features:
        raise ValueError(f"{what} must be CUDA FP16[..., {features}]")
    if t.ndim != 2:
        t = t.reshape(-1, features)
    rows, (stride, column) = t.shape[0], t.stride()
    if column != 1 and features > 1 or rows > 1 and stride < features:
        t, stride = t.contiguous(), features
    return t, rows, stride if rows > 1 else features


def _taken(base, x, ids, adapters):
    """The rows of a call with dense operands, conditions checked at once (a
    call of a few rows is bound by the host); 0 for any other call."""
    k, n = adapters.features
    try:
        shape = ids.shape
        if (base.dtype is torch.float16 and x.dtype is torch.float16 and ids.dtype is torch.int32
                and base.shape == (*shape, n) and x.shape == (*shape, k)
                and base.is_contiguous() and x.is_contiguous() and ids.is_contiguous()
                and base.get_device() == x.get_device() == ids.get_device() == adapters.down.get_device()):
            return ids.numel()
    except AttributeError:
        pass
    return 0


def _meets(t, rows, features, stride, out):
    """Whether a row of `t` shares memory with the dense rows of `out`."""
    t0, o0 = t.data_ptr(), out.data_ptr()
    row = max(0, (o0 - t0 - 2 * features) // (2 * stride) + 1)   # the first that ends behind out's start
    return row < rows and t0 + 2 * stride * row < o0 + 2 * rows * features


def add(base, x, adapters, ids, out=None):
    """base[..., N] plus each row's adapter update of x[..., K]; a new FP16
    tensor, or `out` (`base` itself, or memory that base does not overlap).
    `ids` int32[...] names each row's adapter: negative, or not below the set's
    count, for none (the row is copied).  Rows with the same adapter cost least
    side by side."""
    if not isinstance(adapters, AdapterSet):
        raise ValueError("adapters must be an AdapterSet")
    k, n = adapters.features
    rows = _taken(base, x, ids, adapters)
    if rows:
        b2, x2, bs, xs = base, x, n, k
    else:
        b2, rows, bs = _rows(base, n, "base")
        x2, xrows, xs = _rows(x, k, "x")
        if rows != xrows or base.shape[:-1] != x.shape[:-1]:
            raise ValueError("base and x must have the same rows")
        if not isinstance(ids, torch.Tensor) or ids.dtype != torch.int32 or ids.shape != base.shape[:-1]:
            raise ValueError("ids must be int32, one for each row")
        if any(t.device != base.device for t in (x, ids, adapters.down)):
            raise ValueError("Adapter operands must share one device")
        ids = ids.contiguous()
    if out is None:
        out = torch.empty_like(base, memory_format=torch.contiguous_format)
    elif (not isinstance(out, torch.Tensor) or out.dtype != torch.float16 or out.shape != base.shape
          or out.device != base.device or not out.is_contiguous()):
        raise ValueError("out must be contiguous FP16 of base's shape")
    elif rows and (b2.data_ptr() != out.data_ptr() or bs != n) and _meets(b2, rows, n, bs, out):
        raise ValueError("out must be base itself or not overlap it")   # (other rows still read theirs)
    if rows == 0:
        return out
    rank = adapters.rank
    ws_bytes = int(_native.lib().m2r_adapters_workspace(rows, k, n, rank))
    ws = base.new_empty(ws_bytes, dtype=torch.uint8)
    p = _native.ptr
    with _native.device_of(base):
        _native.call("m2r_adapters_add", p(x2), xs, p(b2), bs, p(adapters.down), p(adapters.up), p(adapters.scale),
                     p(ids), p(out), n, rows, k, n, adapters.count, rank, p(ws), ws_bytes,
                     _native.stream_of(base))
    return out
