"""Log probabilities, entropy and the most likely tokens of rows of logits, in plain numpy and 64 bits.

Test infrastructure only.  Ties go to the lowest id, a NaN ranks above all; a row whose largest logit is infinite or a
NaN has NaN for its numbers.  Pinned by hand-worked rows (tests/test_oracle_drafts.py).
"""

from __future__ import annotations

import numpy as np


def token_logprobs(x: np.ndarray, tokens: np.ndarray, top: int) -> tuple[np.ndarray, np.ndarray, np.ndarray, np.ndarray]:
    """x [N, V], tokens [N] -> (logprobs [N], entropy [N], top ids [N, top], their log probabilities)."""
    x = np.asarray(x, dtype=np.float64)
    n, vocab = x.shape
    logp, entropy = np.zeros(n), np.zeros(n)
    ids, best = np.zeros((n, top), dtype=np.int64), np.zeros((n, top))
    for r in range(n):
        row = x[r]
        order = np.lexsort((np.arange(vocab), -np.where(np.isnan(row), 0.0, row), ~np.isnan(row)))
        ids[r] = order[:top]
        m = row.max()
        if np.isfinite(m):
            d = row - m
            e = np.exp(d)
            norm = np.log(e.sum())
            p = d - norm
            entropy[r] = norm - (e[e > 0] * d[e > 0]).sum() / e.sum()
        else:
            p, entropy[r] = np.full(vocab, np.nan), np.nan
        best[r] = p[ids[r]]
        t = int(tokens[r])
        logp[r] = 0.0 if t < 0 else np.nan if t >= vocab else p[t]
    return logp, entropy, ids, best
