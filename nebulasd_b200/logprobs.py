"""Log probabilities of logits rows on the GPU: given tokens, entropy, top alternatives.

Stands beside ``accept.greedy_accept`` and takes the same logits: where a
request asks for log probabilities, branches over its likeliest continuations,
or scores a prompt, ``token_logprobs`` gives each row's given token its log
probability and rank, the row's entropy, and the ``num_top`` likeliest tokens,
in one launch and without a host sync.  (The reference keeps only
``torch.argmax`` of these logits,
``swiftLLM/swiftllm/worker/layers/post_layer.py:72``.)
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._workspace import ErrorWords
from .kernels.paged_attn import _raw_stream

MAX_TOP = 32  # NEB_MAX_TOP_LOGPROBS
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}

_errors = ErrorWords("token_logprobs")


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor | None      # [R] fp32, None without token_ids
    ranks: torch.Tensor | None         # [R] int32, 1 = the largest logit
    entropy: torch.Tensor              # [R] fp32, nats
    top_ids: torch.Tensor | None       # [R, num_top] int32, None when num_top is 0
    top_logprobs: torch.Tensor | None  # [R, num_top] fp32


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor | None = None, num_top: int = 0) -> TokenLogprobs:
    """``logits`` ``[R, vocab]`` (float16, bfloat16 or float32; contiguous rows, any row stride),
    ``token_ids`` int32 ``[R]`` (-1: no token in this row), ``num_top`` up to 32.

    ``logprobs[r] = log_softmax(logits[r])[token_ids[r]]`` (NaN for -1);
    ``ranks[r]`` is 1 plus the number of larger logits (0 for -1); ``entropy`` is
    in nats; ``top_ids`` are the largest logits' tokens, largest first, ties by
    the lowest id.  Sums are fp32.  Banned tokens (-inf) have probability 0; a
    row with a NaN, a +inf or nothing but -inf gets NaN results.  A token
    outside ``[-1, vocab)`` counts as -1 and is reported by ``workspace_errors``
    (bit 6).  No gradients.  Runs on the current stream of the logits' device; its first call on
    a device must come before any graph capture.
    """
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise ValueError("logits must be a [rows, vocab] tensor of float16, bfloat16 or float32")
    rows, vocab = logits.shape
    index = logits.get_device()
    if index < 0:
        raise ValueError("logits must be on a CUDA device")
    if not 0 < vocab <= 1 << 30 or rows >= 1 << 31:
        raise ValueError("logits need 1 to 2^30 logits per row and fewer than 2^31 rows")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits must have contiguous rows")
    if token_ids is not None:
        if (token_ids.dtype != torch.int32 or token_ids.dim() != 1 or token_ids.shape[0] != rows
                or token_ids.get_device() != index or not token_ids.is_contiguous()):
            raise ValueError("token_ids must be a contiguous int32 vector with one token per row, on the logits' device")
    if not 0 <= num_top <= min(MAX_TOP, vocab):
        raise ValueError(f"num_top must be in [0, min({MAX_TOP}, vocab)]")
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _launch(logits, token_ids, num_top, rows, vocab, index)
    return _launch(logits, token_ids, num_top, rows, vocab, index)


def _launch(logits, token_ids, num_top, rows, vocab, index) -> TokenLogprobs:
    dev = logits.device
    logprobs = ranks = top_ids = top_logprobs = None
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    if token_ids is not None:
        logprobs = torch.empty_like(entropy)
        ranks = torch.empty_like(token_ids)
    if num_top:
        top_logprobs = torch.empty((rows, num_top), dtype=torch.float32, device=dev)
        top_ids = torch.empty_like(top_logprobs, dtype=torch.int32)
    rc = _lib.lib.neb_token_logprobs(
        logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), vocab, rows, _lib.ptr(token_ids), num_top,
        _lib.ptr(logprobs), _lib.ptr(ranks), entropy.data_ptr(), _lib.ptr(top_ids), _lib.ptr(top_logprobs),
        _errors.word(index).data_ptr(), _raw_stream(index))
    _lib.check(rc, "token_logprobs")
    return TokenLogprobs(logprobs, ranks, entropy, top_ids, top_logprobs)


def workspace_errors(device: torch.device | None = None) -> int:
    """Synchronise the device's current stream and return (and clear) the error bits that
    calls on it recorded (bit 6: a token outside ``[-1, vocab)``; bit 3: a bounded
    wait gave up, and its row was read again, slowly)."""
    return _errors.read(device)
