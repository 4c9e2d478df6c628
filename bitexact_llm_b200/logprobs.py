"""Log probabilities of the tokens that a model gave or was given: log p, entropy, rank and the best alternatives of rows of logits,
in one pass (`bx_log_probs`). Takes what every engine's `logits` returns (int64 fixed point) and float logits alike.

`vllm_plugin.rl.int_logp` beside it is the integer-defined log p of the given token alone, for hashes and replays; this one is in
32-bit floats and answers what a serving interface is asked for (token log probabilities with top alternatives)."""

from typing import NamedTuple, Optional

import torch

from . import _native as nv

MAX_TOP = 32
MASKED = -(1 << 62)             # int64 logits of at most this are masked
KINDS = {torch.int64: 0, torch.float32: 1, torch.bfloat16: 2}


class LogProbs(NamedTuple):
    logp: Optional[torch.Tensor]        # float32 [n]: ln p of the given tokens
    entropy: torch.Tensor               # float32 [n]
    rank: Optional[torch.Tensor]        # int64 [n]: 1 for the best token
    top_ids: torch.Tensor               # int64 [n, top]
    top_logp: torch.Tensor              # float32 [n, top]


def log_probs(logits, tokens=None, top=0, fr=24):
    """logits [n, V] (unit column stride): int64 at `fr` fractional bits, float32 or bfloat16; -infinity (int64: at most MASKED) is
    masked. tokens int64 [n] or None; top: alternatives per row, at most MAX_TOP.

    Equal logits go by index. A token outside the vocabulary has logp NaN and rank 0; a row with fewer than `top` unmasked
    entries ends in (-1, -inf); one with NaN or +inf, or without any unmasked entry, is NaN throughout. No host synchronisation."""
    if logits.dim() != 2 or logits.dtype not in KINDS:
        raise ValueError("log_probs: logits [n, V] in int64, float32 or bfloat16")
    n, V = logits.shape
    if V < 1 or V > 1 and logits.stride(1) != 1 or n > 1 and logits.stride(0) < V:
        raise ValueError("log_probs: rows of at least one logit, each contiguous, that do not overlap")
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.shape != (n,)):
        raise ValueError("log_probs: tokens int64 [n], one for each row")
    if not 0 <= top <= MAX_TOP or not 0 <= fr <= 40:
        raise ValueError(f"log_probs: top is 0 .. {MAX_TOP}, fr 0 .. 40")
    nv.here(logits, tokens)
    dev, given = logits.device, tokens is not None
    tokens = tokens.contiguous() if given else None
    # the outputs are parts of two buffers: an allocation each costs more than a small call
    logp, entropy, top_logp = torch.empty(2 * n + n * top, dtype=torch.float32, device=dev).split_with_sizes((n, n, n * top))
    rank, top_ids = torch.empty(n + n * top, dtype=torch.int64, device=dev).split_with_sizes((n, n * top))
    rc = nv.lib().bx_log_probs(KINDS[logits.dtype], logits.data_ptr(), logits.stride(0) if n > 1 else V, nv.ptr(tokens), top, logp.data_ptr(),
                               entropy.data_ptr(), rank.data_ptr(), top_ids.data_ptr(), top_logp.data_ptr(), n, V, fr, nv.stream())
    nv.check(rc, "bx_log_probs")
    return LogProbs(logp if given else None, entropy, rank if given else None, top_ids.view(n, top), top_logp.view(n, top))
