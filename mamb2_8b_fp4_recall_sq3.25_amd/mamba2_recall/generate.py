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

All prompts of a call have the same length.
"""
from __future__ import annotations

import torch

from . import sampling


@torch.no_grad()
def generate(controller, lm_head, prompt, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Continue `prompt` int64[batch,tokens] by as many tokens as `uniforms`
    FP32[batch,new] has columns; returns (ids int64[batch,new], log
    probabilities FP32[batch,new]).  The filters are sampling.sample's: numbers,
    or a value for each request.  The controller's request is reset first and
    stands after the last token but one."""
    if (not isinstance(uniforms, torch.Tensor) or uniforms.ndim != 2 or uniforms.dtype != torch.float32
            or uniforms.shape[1] < 1):
        raise ValueError("uniforms must be FP32[batch,new] with at least one new token")
    if not isinstance(prompt, torch.Tensor) or prompt.ndim != 2 or prompt.shape[0] != uniforms.shape[0]:
        raise ValueError("prompt must be [batch,tokens] with a row for each row of uniforms")
    sampling.filters(uniforms, temperature, top_k, top_p, min_p)   # refused before the request is reset
    hidden = controller.backbone(prompt, reset=True)
    columns = uniforms.t().contiguous()
    ids, logprobs = [], []
    for step in range(columns.shape[0]):
        if step:
            # a row whose logits hold nothing to draw (-1) goes on with token 0
            hidden = controller.backbone(ids[-1].clamp(min=0)[:, None])
        token, logprob = sampling.sample(lm_head(hidden[:, -1]), columns[step], temperature=temperature, top_k=top_k,
                                         top_p=top_p, min_p=min_p)
        ids.append(token)
        logprobs.append(logprob)
    return torch.stack(ids, 1), torch.stack(logprobs, 1)
