"""Scores of tokens that were generated, drafted or given, from rows of logits.

``token_logprobs`` returns, for each row of logits and the token that belongs
to it, the token's log probability, the entropy of the row's distribution and
the most likely tokens with their log probabilities. With x a row,

    m = max x,  S = sum_v e^(x_v - m),  ln p_v = (x_v - m) - ln S,
    entropy = -sum_v p_v ln p_v = ln S - sum_v (x_v - m) e^(x_v - m) / S

in fp32 whatever the type of the logits. The reference project has no
counterpart (its engine returns token ids only). CUDA tensors only.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L
from .fp8 import _call

MAX_TOP = 32

_DT = {torch.float32: L.NPL_F32, torch.float16: L.NPL_F16, torch.bfloat16: L.NPL_BF16}
_empty = torch.empty_strided
_token_logprobs = L.lib.npl_token_logprobs


class TokenLogprobs(NamedTuple):
    """Results for logits [..., V]: fp32 and int64 tensors."""
    logprobs: torch.Tensor      # [...]: ln p of the given token; 0 where its id is -1
    entropy: torch.Tensor       # [...]: of the row's distribution, in nats
    top_ids: torch.Tensor       # [..., top_k]: the most likely tokens, of equal ones the lowest first
    top_logprobs: torch.Tensor  # [..., top_k]


def _same_device(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    d = first.get_device()
    if d < 0:
        raise ValueError("the log probabilities run on CUDA tensors only")
    for t in others:
        if t is not None and t.get_device() != d:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Logits fp16, bf16 or fp32 [..., V] (as the runner returns them) and the
    tokens int64 [...] -> TokenLogprobs. A token of -1 marks a padding row,
    whose log probability is given as 0; an id outside the vocabulary gives NaN
    and is recorded in the device status word (``_lib.device_status``). Logits
    of minus infinity (tokens that a sampler has barred) have probability 0; a
    row of nothing else, or one that holds a NaN or plus infinity, gives NaN.
    ``top_k`` is 0 to 32. Runs on the current stream of the logits' device,
    keeps no workspace and can be captured into a CUDA graph."""
    _same_device(logits, token_ids)
    dt = _DT.get(logits.dtype)
    if dt is None:
        raise ValueError("logits must be one of float32, float16, bfloat16")
    if logits.dim() == 0 or logits.size(-1) == 0:
        raise ValueError("logits need at least one column")
    shape = logits.shape
    lead, v = shape[:-1], shape[-1]
    if token_ids.dtype is not torch.int64 or token_ids.shape != lead:
        raise ValueError("token_ids must be int64 with the shape of the logits without their last dimension")
    if not 0 <= top_k <= min(MAX_TOP, v):
        raise ValueError(f"top_k must be 0 to {MAX_TOP}, and no more than the vocabulary")
    x = logits if len(shape) == 2 else logits.reshape(-1, v)
    n, ld = (shape if len(shape) == 2 else x.shape)[0], v
    if not x.is_contiguous():
        ld, one = x.stride()
        if (v > 1 and one != 1) or (n > 1 and ld < v):
            x, ld = x.contiguous(), v
    ids = token_ids.contiguous()
    dev = logits.device
    lp, entropy = _empty((n,), (1,), dtype=torch.float32, device=dev), _empty((n,), (1,), dtype=torch.float32, device=dev)
    top_ids = _empty((n, top_k), (top_k, 1), dtype=torch.int64, device=dev)
    top_lp = _empty((n, top_k), (top_k, 1), dtype=torch.float32, device=dev)
    if n:
        _call(_token_logprobs, dev, x.data_ptr(), dt, ld, n, v, ids.data_ptr(), top_k, lp.data_ptr(),
              entropy.data_ptr(), top_ids.data_ptr(), top_lp.data_ptr())
    if len(shape) != 2:
        lp, entropy = lp.view(lead), entropy.view(lead)
        top_ids, top_lp = top_ids.view(*lead, top_k), top_lp.view(*lead, top_k)
    return TokenLogprobs(lp, entropy, top_ids, top_lp)
