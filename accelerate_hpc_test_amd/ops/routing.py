"""Routing to experts: which experts a token goes to and with what weights, from the router's logits, with the logits'
gradient (`models/moe.py` calls it for every form beyond the plain softmax top-k). GPU tensors run
`csrc/kernels/route_experts.hip`, one launch forward and one backward; CPU tensors run the PyTorch reference below.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from ._ext import ext, forward_mode, use_native
from .fused import ROW_DTYPES

MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 64, 64  # of the HIP kernel
# the sigmoid of a logit below this is 0 in the type: half the smallest number, 2^-150 or 2^-1075
_NO_SCORE = {torch.float32: -150 * math.log(2), torch.float64: -1075 * math.log(2)}


def route_experts_reference(logits, top_k, scoring="softmax", bias=None, n_groups=1, topk_groups=1, renormalize=True, scale=1.0):
    x = logits if logits.dtype == torch.float64 else logits.float()
    T, E = x.shape
    score = torch.softmax(x, -1) if scoring == "softmax" else torch.sigmoid(x)
    with torch.no_grad():
        if bias is None and topk_groups == n_groups:
            key = x.double()  # the scores' own order
        else:  # sums of scores and a bias, in 64 bits: the order must not hang on a rounding
            key = torch.softmax(x.double(), -1) if scoring == "softmax" else torch.sigmoid(x.double())
            if bias is not None:
                key = key + bias.double()
        key = torch.where(key.isnan(), torch.full_like(key, -math.inf), key)
        if topk_groups < n_groups:
            size = E // n_groups
            rating = torch.topk(key.view(T, n_groups, size), min(2, size), dim=-1)[0].sum(-1)
            best = torch.sort(rating, dim=-1, descending=True, stable=True)[1][:, :topk_groups]
            closed = torch.ones_like(rating, dtype=torch.bool).scatter_(1, best, False)
            # closed experts sort behind every open one, -inf among them
            order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
            shut = closed.repeat_interleave(size, 1).gather(1, order)
            ids = order.gather(1, torch.sort(shut.to(torch.int8), dim=-1, stable=True)[1])[:, :top_k]
        else:
            ids = torch.sort(key, dim=-1, descending=True, stable=True)[1][:, :top_k]
    if not renormalize:
        return score.gather(1, ids) * scale, ids
    # Shares in logarithms: the chosen scores may lie any distance below the largest. Scores that are all zero share nothing.
    v = x.gather(1, ids)
    top = v.detach().amax(-1, keepdim=True)
    none = top == -math.inf if scoring == "softmax" else top < _NO_SCORE[x.dtype]
    v = torch.where(none, torch.zeros_like(v), v)
    w = torch.softmax(v if scoring == "softmax" else torch.nn.functional.logsigmoid(v), -1)
    w = torch.where(none, torch.zeros_like(w), w)
    if scoring == "softmax":  # a row without a distribution
        w = torch.where(score.detach().sum(-1, keepdim=True).isnan(), torch.full_like(w, math.nan), w)
    return w * scale, ids


def route_experts(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
                  n_groups: int = 1, topk_groups: int = 1, renormalize: bool = True, scale: float = 1.0):
    """The `top_k` experts of each token and their weights from router logits [T, E] (bf16, fp16 or fp32).

    Scores are softmax(logits) or sigmoid(logits) (`scoring`). Experts are chosen by score + `bias` ([E], optional, in 32 bits: it
    steers the choice alone, balances the load, and gets no gradient), within the `topk_groups` of `n_groups` equal groups whose two
    best keys have the largest sum; equal keys go to the lower index, keys are compared in 64 bits. Weights are the chosen scores,
    divided by their sum (`renormalize`; scores that are all 0 in 32 bits give 0), times `scale` (2^-60 to 2^60 in size). Returns
    (weights fp32 [T, k], experts int64 [T, k]) in falling order of the keys; the weights are differentiable with respect to the
    logits, on a GPU once."""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"route_experts: logits must be [tokens, experts], got shape {tuple(logits.shape)}")
    if not logits.is_floating_point():
        raise TypeError(f"route_experts: logits must be of a floating type, got {logits.dtype}")
    E = logits.shape[1]
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"route_experts: scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    if n_groups < 1 or E % n_groups or not 1 <= topk_groups <= n_groups:
        raise ValueError(f"route_experts: {topk_groups} of {n_groups} groups over {E} experts")
    if not 1 <= top_k <= E // n_groups * topk_groups:
        raise ValueError(f"route_experts: top_k={top_k} of {E // n_groups * topk_groups} experts within reach")
    if not 2.0**-60 <= abs(scale) <= 2.0**60:  # shares down to 2^-60 and gradients up to 2^60 stay within 32 bits
        raise ValueError(f"route_experts: scale must be between 2^-60 and 2^60 in size, got {scale}")
    if bias is not None:
        if bias.shape != (E,) or bias.device != logits.device:
            raise ValueError(f"route_experts: bias must be a [{E}] tensor on the logits' device")
        bias = bias.detach() if logits.dtype == torch.float64 else bias.detach().float()
    if not (use_native(logits) and logits.dtype in ROW_DTYPES) or forward_mode(logits):
        return route_experts_reference(logits, top_k, scoring, bias, n_groups, topk_groups, renormalize, scale)
    if E > MAX_EXPERTS or top_k > MAX_TOP_K or n_groups > MAX_GROUPS:
        raise ValueError(f"HIP route_experts takes at most {MAX_EXPERTS} experts, {MAX_TOP_K} choices and {MAX_GROUPS} groups "
                         f"(got {E}, {top_k}, {n_groups})")
    if bias is not None:
        bias = bias.contiguous()
    w, ids = ext().route_experts(logits, top_k, scoring == "softmax", bias, n_groups, topk_groups, renormalize, scale)
    return w, ids
