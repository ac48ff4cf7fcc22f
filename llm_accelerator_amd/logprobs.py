"""Log probabilities of given tokens, with entropy, rank and the most likely alternatives, out of logits.

No counterpart in the reference, whose only answer is the argmax
(``10_validate_full_run_one_token.py:52-56``); :func:`token_logprobs` takes the logits that
``run_manual_one_token``, ``BatchedDecoder.step``, ``Prefill.run`` or ``mx_linear`` leave.  It is
launched on torch's current stream of the logits' device, does not synchronise, keeps nothing between
calls and can be captured into a graph.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._lib import Q4D_BF16, Q4D_F16, Q4D_F32
from .model import call_on

MAX_TOP = 32
MAX_VOCAB = 1 << 20
SMALL_WORKSPACE = 1 << 15  # bytes that the results may keep alive beside them
_DTYPES = {torch.float16: Q4D_F16, torch.bfloat16: Q4D_BF16, torch.float32: Q4D_F32}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor | None  # fp32 [...]: of the given tokens
    rank: torch.Tensor | None     # int32 [...]: how many tokens come before them (0: the most likely)
    entropy: torch.Tensor         # fp32 [...]: of the distributions (natural logarithm)
    top_logprobs: torch.Tensor    # fp32 [..., top]
    top_ids: torch.Tensor         # int32 [..., top]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, top: int = 0) -> TokenLogprobs:
    """Of ``logits`` [..., vocab] (fp32, fp16 or bf16; rows may be slices of longer ones) the log
    probability and rank of ``targets`` [...] (int32; ``None``: neither), the entropy, and the ``top``
    most likely tokens (0 .. 32).  Tokens are ordered by logit, equal ones by index, the lowest first.

    Up to 2^23 rows (x ceil(vocab / 16384)).  A token of -Inf (a masked one) has the probability 0.  A target
    outside the vocabulary (a padded row's) gives NaN and rank -1.  A row with nothing but -Inf, or with NaN or
    +Inf, has NaN for log probabilities and entropy; NaN comes last in the order."""
    if not logits.is_cuda:
        raise ValueError("logits must be a GPU tensor (libq4dec has no CPU path)")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be fp32, fp16 or bf16, got {logits.dtype}")
    if logits.dim() == 0 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"logits must be [..., vocab], vocab 1 .. {MAX_VOCAB}, got {tuple(logits.shape)}")
    lead, vocab, index = logits.shape[:-1], logits.shape[-1], logits.get_device()
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 .. {min(MAX_TOP, vocab)}, got {top}")
    if targets is not None:
        if targets.dtype != torch.int32 or targets.shape != lead or targets.get_device() != index:
            raise ValueError(f"targets must be int32 {tuple(lead)} on {logits.device}")
        targets = targets.contiguous()
    x = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    rows, step, have = x.shape[0], x.stride(0), targets is not None
    if rows * -(-vocab // 16384) > 1 << 23:
        raise ValueError(f"rows x ceil(vocab / 16384) must be at most 2^23, got {tuple(logits.shape)}")
    if (vocab > 1 and x.stride(1) != 1) or (rows > 1 and step < vocab):
        x, step = x.contiguous(), vocab
    nbytes = _lib.load().q4d_token_logprobs_workspace_bytes(rows, vocab, top) if rows else 0
    # the results lie side by side in one allocation, behind the workspace if that is small
    inside = (nbytes + 3) // 4 if nbytes <= SMALL_WORKSPACE else 0
    got = x.new_empty(inside + rows * (3 + 2 * top), dtype=torch.float32)
    _, logprob, entropy, rank, top_logprobs, top_ids = got.split((inside, rows, rows, rows, rows * top, rows * top))
    if rows:
        ws = got if inside else x.new_empty(nbytes, dtype=torch.uint8)
        at, size = got.data_ptr() + 4 * inside, 4 * rows
        call_on(index, "q4d_token_logprobs", x.data_ptr(), _DTYPES[x.dtype], step, rows, vocab,
                targets.data_ptr() if have else None, top, at if have else None, at + 2 * size if have else None, at + size,
                at + 3 * size if top else None, at + (3 + top) * size if top else None, ws.data_ptr(), nbytes)
    if len(lead) != 1:
        logprob, entropy, rank = logprob.view(lead), entropy.view(lead), rank.view(lead)
    wide = (*lead, top)
    return TokenLogprobs(logprob if have else None, rank.view(torch.int32) if have else None, entropy, top_logprobs.view(wide), top_ids.view(torch.int32).view(wide))


__all__ = ["TokenLogprobs", "token_logprobs", "MAX_TOP", "MAX_VOCAB"]
