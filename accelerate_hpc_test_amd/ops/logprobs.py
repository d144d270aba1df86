"""Log-probabilities of given tokens, the entropy of their distributions and the best alternatives, with gradients: what
preference, policy and distillation losses read from a language model's logits. GPU tensors run
`csrc/kernels/token_logprobs.hip` (the logits are read once forward, read once and their gradient written once backward; no
[rows, vocabulary] tensor of probabilities exists); CPU tensors run the PyTorch reference below.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from ._ext import ext, forward_mode, use_native
from .fused import ROW_DTYPES

MAX_TOP_K = 64  # alternatives per row on a GPU


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # fp32 [...]
    entropy: torch.Tensor  # fp32 [...]
    top_logprobs: Optional[torch.Tensor]  # fp32 [..., top_k], falling; None without alternatives
    top_tokens: Optional[torch.Tensor]  # int64 [..., top_k]; equal logits: the lower token first


def token_logprobs_reference(logits, tokens, top_k=0, temperature=1.0, ignore_index=-100):
    counts = tokens != ignore_index
    acc = logits if logits.dtype == torch.float64 else logits.float()
    acc = torch.where(counts.unsqueeze(-1), acc, torch.zeros_like(acc))  # ignored rows are not read: they may hold anything
    named = (tokens >= 0) & (tokens < logits.shape[-1])
    z = acc / temperature
    logp = torch.log_softmax(z, dim=-1)
    zero = torch.zeros((), dtype=logp.dtype, device=logp.device)
    at = torch.where(named, tokens, torch.zeros_like(tokens)).unsqueeze(-1)
    lp = logp.gather(-1, at).squeeze(-1)
    lp = torch.where(named, lp, torch.full_like(lp, math.nan))
    p = logp.exp()
    gone = p == 0  # p log p is 0 there
    entropy = -(p * logp.masked_fill(gone, 0.0)).masked_fill(gone, 0.0).sum(-1)
    top_lp = top_id = None
    if top_k:
        sound = ~entropy.detach().isnan().unsqueeze(-1)
        top_id = torch.sort(acc.detach(), dim=-1, descending=True, stable=True)[1][..., :top_k]
        top_lp = torch.where(counts.unsqueeze(-1), logp.gather(-1, top_id), zero)
        top_id = torch.where(counts.unsqueeze(-1) & sound, top_id, torch.full_like(top_id, -1))
    return TokenLogprobs(torch.where(counts, lp, zero), torch.where(counts, entropy, zero), top_lp, top_id)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """log softmax(logits / temperature) at `tokens`, the entropy of that distribution, and its `top_k` best alternatives.

    logits [..., V] in bf16, fp16 or fp32; tokens: integers [...]; temperature: 2^-100 to 2^100. All outputs are fp32 and differentiable with respect to the
    logits (the alternatives at their chosen tokens). Rows whose token is `ignore_index` give 0, 0, 0 and -1 and no gradient;
    a token outside [0, V) gives a NaN log-probability that carries no gradient. The backward reads the logits again: beside
    `cross_entropy` on the same logits, give that `inplace_backward=False`. Logits of -inf are impossible tokens: probability 0,
    nothing added to the entropy. A row with NaN or +inf, or of -inf alone, has no distribution: NaN, and -1 for the alternatives."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"token_logprobs: logits must be [..., vocabulary], got shape {tuple(logits.shape)}")
    V = logits.shape[-1]
    if tokens.shape != logits.shape[:-1] or tokens.device != logits.device:
        raise ValueError(f"token_logprobs: tokens must be {tuple(logits.shape[:-1])} on the logits' device, got {tuple(tokens.shape)}")
    if not logits.is_floating_point():
        raise TypeError(f"token_logprobs: logits must be of a floating type, got {logits.dtype}")
    if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
        raise TypeError(f"token_logprobs: tokens must be integers, got {tokens.dtype}")
    if not 0 <= top_k <= V:
        raise ValueError(f"token_logprobs: top_k must be within the vocabulary ({top_k} of {V})")
    if not 2.0**-100 <= temperature <= 2.0**100:  # its quotient with any logit difference that counts is held in 32 bits
        raise ValueError(f"token_logprobs: temperature must be within 2^-100 and 2^100, got {temperature}")
    tokens = tokens.to(torch.int64)
    if not (use_native(logits) and logits.dtype in ROW_DTYPES) or forward_mode(logits):
        return token_logprobs_reference(logits, tokens, top_k, temperature, ignore_index)
    if top_k > MAX_TOP_K:
        raise ValueError(f"HIP token_logprobs gives at most {MAX_TOP_K} alternatives (got top_k={top_k})")
    out = ext().token_logprobs(logits, tokens, top_k, 1.0 / temperature, ignore_index)
    return TokenLogprobs(*out) if top_k else TokenLogprobs(*out, None, None)
