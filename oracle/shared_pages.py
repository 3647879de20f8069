"""Forked sequences on shared pages, in plain numpy: test infrastructure only.

Policies (this project's own: the reference copies its tensors): a fork shares the
source's whole pages and copies the begun one into a page popped from the stack,
forks in order; refs[p] counts a page's holders beyond the first; a release pushes
a page when its last holder leaves, in the order ascending sequence, last logical
page first, at the last place among holders that leave together; a compaction moves
a page once.  Pinned by hand-worked cases and by ownership invariants
(tests/test_oracle_shared_pages.py).
"""

from __future__ import annotations

import numpy as np

from oracle import reference_cpu as ref


def fork(stack: np.ndarray, top: int, refs: np.ndarray, block_table: np.ndarray, seq_lens: np.ndarray, src: list[int],
         dst: list[int], block: int, pools: list) -> int:
    """Returns the new top of the stack."""
    for s, d in zip(src, dst):
        n = int(seq_lens[s])
        for j in range(n // block):
            block_table[d, j] = block_table[s, j]
            refs[block_table[s, j]] += 1
        if n % block:
            top -= 1
            block_table[d, n // block] = stack[top]
            for p in pools:
                p[int(stack[top])] = p[int(block_table[s, n // block])]
        seq_lens[d] = n
    return top


def release(stack: np.ndarray, top: int, refs: np.ndarray, block_table: np.ndarray, seq_lens: np.ndarray,
            mask: np.ndarray, block: int) -> int:
    """Returns the new top of the stack."""
    for b in np.flatnonzero(mask):
        for j in range(-(-int(seq_lens[b]) // block) - 1, -1, -1):
            p = int(block_table[b, j])
            if refs[p] == 0:
                stack[top] = p
                top += 1
            else:
                refs[p] -= 1
            block_table[b, j] = -1
        seq_lens[b] = 0
    return top


def compact(pools: list, refs: np.ndarray, block_table: np.ndarray, seq_lens: np.ndarray,
            block: int) -> tuple[np.ndarray, int, int]:
    """As ref.compact (stack, top, pages moved), the counts moving with their pages."""
    movers, holes, _ = ref.compact_plan(block_table, seq_lens, block, pools[0].shape[0])
    refs[holes] = refs[movers]
    refs[movers] = 0
    return ref.compact(pools, block_table, seq_lens, block)


def check(refs: np.ndarray, stack: np.ndarray, top: int, block_table: np.ndarray, seq_lens: np.ndarray,
          block: int) -> None:
    """Every page is free once, or held by 1 + refs sequences; a page that is not whole by one."""
    held = np.zeros(refs.shape[0], dtype=np.int64)
    for b in range(block_table.shape[0]):
        n = int(seq_lens[b])
        for j in range(-(-n // block)):
            p = int(block_table[b, j])
            held[p] += 1
            if (j + 1) * block > n:
                assert refs[p] == 0, f"page {p}, begun by sequence {b}, is shared"
    free = np.bincount(stack[:top], minlength=refs.shape[0])
    assert ((held > 0) ^ (free == 1)).all() and (free <= 1).all()
    assert (refs == np.maximum(held - 1, 0)).all()
