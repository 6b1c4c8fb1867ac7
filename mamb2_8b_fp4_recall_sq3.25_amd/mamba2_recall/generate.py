"""Generation for a batch of requests through an installed controller: the
prompt in one backbone call, then one token at a time, each drawn on the
device from given uniform numbers (reference: the greedy loop of
scripts/infer_fp4_ridge_resurface_v1.py:100-110, which asks the host for every
token).  Works with any controller; full_state.FullState takes prompts at
matrix rate, and controller.use_adapters gives every request its own adapter:

    sets = [{"in_proj": adapters.AdapterSet(down, up, scale)}     # for each layer
            for down, up, scale in weights]
    with full_state.FullState(model) as controller:               # installed while it runs
        controller.use_adapters(sets, ids)                        # int32[batch], -1 for none
        new, logprobs = generate.generate(controller, lm_head, prompt, uniforms,
                                          temperature=0.8, top_k=50, top_p=0.95)

A queue of prompts of different lengths is padded on the right and goes in one
call through full_state.FullState; its projections and the head may be in 8-bit
integers (int8), and each request may have penalties, biases and a grammar of
its own.
"""
from __future__ import annotations

import torch

from . import sampling


@torch.no_grad()
def generate(controller, lm_head, prompt, uniforms, *, lengths=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
             repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
    """Continue `prompt` int64[batch,tokens] by as many tokens as `uniforms`
    FP32[batch,new] has columns; returns (ids int64[batch,new], log
    probabilities FP32[batch,new]).  The filters are sampling.sample's, the
    penalties, bias and masks sampling.adjust's: numbers, or a value for each
    request.  `allowed` is the masks for all steps, or a function of the ids
    drawn so far, int64[batch,step], that gives the next step's, or None.
    `lengths` int32[batch] (a controller that takes it): the tokens of each
    prompt, at least one; those behind them, of any value, count for nothing.
    The controller's request is reset first and stands after the last token
    but one."""
    if (not isinstance(uniforms, torch.Tensor) or uniforms.ndim != 2 or uniforms.dtype != torch.float32
            or uniforms.shape[1] < 1):
        raise ValueError("uniforms must be FP32[batch,new] with at least one new token")
    if not isinstance(prompt, torch.Tensor) or prompt.ndim != 2 or prompt.shape[0] != uniforms.shape[0]:
        raise ValueError("prompt must be [batch,tokens] with a row for each row of uniforms")
    # refused before the request is reset; what needs the vocabulary (the width of masks) and what a function of
    # masks gives, when it meets the logits
    sampling.filters(uniforms, temperature, top_k, top_p, min_p)
    sampling.penalties(uniforms, repetition, presence, frequency)
    sampling.biases(uniforms, bias)
    batch, new = uniforms.shape
    if lengths is not None and (not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32
                                or tuple(lengths.shape) != (batch,) or lengths.device != uniforms.device):
        raise ValueError("lengths must be int32[batch] on the device of uniforms")
    if not callable(allowed):
        if allowed is not None and not isinstance(allowed, torch.Tensor):
            raise ValueError("allowed must be a tensor of masks or a function that gives them")
        sampling.masks(uniforms, None, allowed, None)
    counted = any(isinstance(v, torch.Tensor) or v != d for v, d in ((repetition, 1), (presence, 0), (frequency, 0)))
    if counted:
        sampling._list(prompt, lengths, "prompt", batch, uniforms.get_device())
    if lengths is None:
        last = controller.backbone(prompt, reset=True)[:, -1]
    else:
        hidden = controller.backbone(prompt, reset=True, lengths=lengths)
        at = lengths.long().clamp(1, prompt.shape[1]) - 1
        last = hidden[torch.arange(batch, device=hidden.device), at]
    columns = uniforms.t().contiguous()
    ids, logprobs = torch.empty((batch, new), dtype=torch.int64, device=uniforms.device), []
    for step in range(new):
        drawn = ids[:, :step]
        if step:
            # a row whose logits hold nothing to draw (-1) goes on with token 0
            last = controller.backbone(drawn[:, -1:].clamp(min=0))[:, -1]
        logits = lm_head(last)
        masks = allowed(drawn) if callable(allowed) else allowed
        if counted or bias is not None or masks is not None:
            logits = sampling.adjust(logits, prompt=prompt if counted else None,
                                     prompt_lengths=lengths if counted else None,
                                     tokens=drawn if counted and step else None, repetition=repetition,
                                     presence=presence, frequency=frequency, bias=bias, allowed=masks)
        token, logprob = sampling.sample(logits, columns[step], temperature=temperature, top_k=top_k, top_p=top_p,
                                         min_p=min_p)
        ids[:, step] = token
        logprobs.append(logprob)
    return ids, torch.stack(logprobs, 1)
