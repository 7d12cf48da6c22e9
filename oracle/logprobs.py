"""Restatement of a row's log probabilities in 64 bits (CPU).

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

The reference has no counterpart; this follows the definitions: ``log p_j = x_j -
log(sum_i exp(x_i))``, rank ``1 + #{j : x_j > x_t}``, entropy ``-sum_j p_j log p_j``
with ``0 log 0 = 0``.  Order: NaN above everything, ties (``-0 == +0``) to the lowest index.
"""
from __future__ import annotations

import math

import numpy as np
import torch


def token_logprobs(logits: torch.Tensor, token_ids=None, num_top: int = 0):
    """``(logprobs, ranks, entropy, top_ids, top_logprobs)`` as numpy arrays (None where not asked for)."""
    x = logits.detach().cpu().double().numpy()
    rows, vocab = x.shape
    lp, rk, ent = np.full(rows, math.nan), np.zeros(rows, np.int64), np.full(rows, math.nan)
    ids, tops = np.zeros((rows, num_top), np.int64), np.full((rows, num_top), math.nan)
    for r in range(rows):
        v = x[r]
        order = np.where(np.isnan(v), math.inf, v)
        # NaN sorts above +inf: a second key tells them apart.
        first = np.lexsort((np.arange(vocab), -order, ~np.isnan(v)))
        ids[r] = first[:num_top]
        m = v.max()
        valid = math.isfinite(m)
        if valid:
            logp = (v - m) - math.log(np.exp(v - m).sum())  # the maximum apart: it may be far from log(vocab)
            p = np.exp(logp)
            ent[r] = -(p[p > 0] * logp[p > 0]).sum()
            tops[r] = logp[ids[r]]
        t = -1 if token_ids is None else int(token_ids[r])
        if 0 <= t < vocab:
            rk[r] = 1 + (0 if np.isnan(v[t]) else int(np.isnan(v).sum() + (v > v[t]).sum()))
            if valid:
                lp[r] = logp[t]
    return (None if token_ids is None else lp, None if token_ids is None else rk, ent,
            ids if num_top else None, tops if num_top else None)
