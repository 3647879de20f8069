"""Drafted tokens in plain numpy: which the model accepts, and the accepted ones kept in the 4-bit pages.

Test infrastructure only.  Node t of a tree is the t-th of a sequence's newest tokens and follows node parents[t] < t
(-1: the tokens before the tree).  Accepted are node 0 and, after an accepted node, the first child whose token is
the model's pick after that node.  Kept tokens move together behind the tokens before the tree, the length is cut
behind them, pages without a token go on the free stack (sequences ascending, last page first).  Pinned by
hand-worked cases (tests/test_oracle_drafts.py).
"""

from __future__ import annotations

import numpy as np

from oracle.fp4_cache import Pages

BADARG, STACK = 4, 8  # SKV_STATUS_*


def accept(parents: np.ndarray, tokens: np.ndarray, picks: np.ndarray,
           n_new: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(path [B, T], n_keep [B], next [B])."""
    batch, t_max = parents.shape
    path, n_keep = np.full((batch, t_max), -1, dtype=np.int32), np.zeros(batch, dtype=np.int32)
    following = np.full(batch, -1, dtype=picks.dtype)
    for b in range(batch):
        n = min(int(n_new[b]), t_max)
        at = 0 if n > 0 else None
        while at is not None:
            path[b, n_keep[b]] = at
            n_keep[b] += 1
            following[b] = picks[b, at]
            children = [t for t in range(at + 1, n) if parents[b, t] == at and tokens[b, t] == picks[b, at]]
            at = children[0] if children else None
    return path, n_keep, following


def keep(stack: np.ndarray, top: int, block_table: np.ndarray, seq_lens: np.ndarray, n_new: np.ndarray, path: np.ndarray,
         n_keep: np.ndarray, pools: list[np.ndarray], refs: np.ndarray | None = None) -> tuple[int, int]:
    """Returns (new top of the stack, status); where the status is not 0 nothing is written."""
    block, n_pages = pools[0].shape[1], stack.shape[0]
    shared = np.zeros(n_pages, dtype=np.int64) if refs is None else refs

    def page(b, j):
        p = int(block_table[b, j])
        return p if 0 <= p < n_pages else None

    moves, freed = [], []
    if not 0 <= top <= n_pages:
        return top, BADARG
    for b in range(block_table.shape[0]):
        length, n, k = int(seq_lens[b]), int(n_new[b]), int(n_keep[b])
        if not (0 <= length <= block_table.shape[1] * block and 0 <= k <= n <= length and k <= path.shape[1]):
            return top, BADARG
        base, steps = length - n, [int(p) for p in path[b, :k]]
        if steps != sorted(set(steps)) or any(not 0 <= p < n for p in steps):
            return top, BADARG
        for i, p in enumerate(steps):
            if p != i:
                src, dst = page(b, (base + p) // block), page(b, (base + i) // block)
                if src is None or dst is None or shared[dst]:
                    return top, BADARG
                moves.append((src, (base + p) % block, dst, (base + i) % block))
        left = base + k
        if left < length:
            for j in range(-(-length // block) - 1, left // block - 1, -1):
                if page(b, j) is None or shared[page(b, j)]:
                    return top, BADARG
                if j >= -(-left // block):
                    freed.append((b, j))
    if top + len(freed) > n_pages:
        return top, STACK
    for pool in pools:
        p = Pages(pool)
        for src, s, dst, d in moves:
            for kv in range(2):
                for have, to in zip(p._at(s, kv), p._at(d, kv)):
                    p.flat[dst, :, to] = p.flat[src, :, have]
    for b, j in freed:
        stack[top] = block_table[b, j]
        block_table[b, j] = -1
        top += 1
    seq_lens -= (n_new - n_keep).astype(seq_lens.dtype)
    return top, 0
