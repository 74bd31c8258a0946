"""Log probabilities of given tokens, entropy and the most likely alternatives from logits.

What a server returns next to a sampled token, and what scoring a prompt needs: one pass
over each row of logits (``pi_token_logprobs``). ``LmHead.logprobs`` chains it to the
resident projection.
"""
from __future__ import annotations

from typing import Any, NamedTuple

import torch

from ._lib import PI_ERR_ARG, PI_QT_BF16, PI_QT_F16, PI_QT_F32, Context, PiError, lib, raw_stream

_DTYPES = {torch.float32: PI_QT_F32, torch.float16: PI_QT_F16, torch.bfloat16: PI_QT_BF16}


class TokenLogprobs(NamedTuple):
    """``token_logprobs``' answer; a part that was not asked for is None."""

    logp: Any  # f32, shaped like targets
    entropy: Any  # f32 [T]
    top_ids: Any  # int32 [T, n_top]
    top_logp: Any  # f32 [T, n_top]


def token_logprobs(logits, targets=None, n_top: int = 0) -> TokenLogprobs:
    """Scores of every row of ``logits`` [T, V] (CUDA f32, f16 or bf16; rows may be strided).

    targets: int64 [T] or [T, K], the tokens to score; a negative one is padding and gets 0.
    A target >= V gives NaN and is reported by ``Context.sync_check`` (PI_ERR_INDEX).
    n_top: 0 to 32 alternatives, most likely first, ties to the lowest id; id -1 and -inf
    where fewer than n_top tokens have a probability above zero.

    A logit of -inf masks its token. A row that is all -inf has entropy 0, log
    probabilities -inf and ids -1; a row with a NaN or +inf gives NaN and ids -1.
    """
    qt = _DTYPES.get(logits.dtype)
    if qt is None or logits.dim() != 2 or not logits.is_cuda:
        raise PiError(PI_ERR_ARG, "logprobs: logits must be a CUDA tensor [T, V] of f32, f16 or bf16")
    (T, V), (ld, step) = logits.shape, logits.stride()
    if V < 1 or (V > 1 and step != 1):
        raise PiError(PI_ERR_ARG, "logprobs: need V >= 1 logits a row, next to one another")
    dev, K, logp = logits.device, 0, None
    if targets is not None:
        if targets.dtype != torch.int64 or targets.device != dev or targets.dim() not in (1, 2) or \
                targets.shape[0] != T:
            raise PiError(PI_ERR_ARG, "logprobs: targets must be int64 [T] or [T, K] on the logits' device")
        targets = targets.contiguous()
        K = 1 if targets.dim() == 1 else targets.shape[1]
        logp = torch.empty_like(targets, dtype=torch.float32)
    entropy = torch.empty(T, dtype=torch.float32, device=dev)
    ids = top = None
    if n_top:
        if not 0 < n_top <= 32:
            raise PiError(PI_ERR_ARG, "logprobs: 0 <= n_top <= 32")
        ids = torch.empty(T, n_top, dtype=torch.int32, device=dev)
        top = torch.empty(T, n_top, dtype=torch.float32, device=dev)
    if T:
        ctx = Context.of(dev.index)
        rc = lib().pi_token_logprobs(ctx.h, logits.data_ptr(), qt, T, V, ld, targets.data_ptr() if K else None, K,
                                     n_top, logp.data_ptr() if K else None, entropy.data_ptr(),
                                     ids.data_ptr() if n_top else None, top.data_ptr() if n_top else None,
                                     raw_stream(dev.index))
        if rc:
            ctx.check(rc)
    return TokenLogprobs(logp, entropy, ids, top)
