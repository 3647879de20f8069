"""The oracle of forked sequences: a case by hand, and ownership over random histories."""

from __future__ import annotations

import numpy as np
import torch

from oracle import reference_cpu as ref
from oracle import shared_pages as ora


def test_fork_and_release_by_hand() -> None:
    stack, top = ref.free_stack_init(6)
    refs, bt, lens = np.zeros(6, np.int32), np.full((3, 3), -1, np.int32), np.zeros(3, np.int32)
    pool = torch.arange(6)[:, None].repeat(1, 4)
    _, top = ref.reserve(stack, top, bt, lens, np.array([9, 0, 0]), 4)
    assert bt[0].tolist() == [0, 1, 2] and top == 3
    top = ora.fork(stack, top, refs, bt, lens, [0, 0], [1, 2], 4, [pool])
    assert bt.tolist() == [[0, 1, 2], [0, 1, 3], [0, 1, 4]] and refs.tolist() == [2, 2, 0, 0, 0, 0] and top == 1
    assert pool[3:5].tolist() == [[2] * 4, [2] * 4]
    top = ora.release(stack, top, refs, bt, lens, np.array([1, 0, 1]), 4)
    assert refs.tolist() == [0] * 6 and stack[:top].tolist() == [5, 2, 4] and bt[1].tolist() == [0, 1, 3]
    top = ora.release(stack, top, refs, bt, lens, np.array([0, 1, 0]), 4)
    assert stack[:top].tolist() == [5, 2, 4, 3, 1, 0]


def test_ownership_over_random_histories() -> None:
    rng = np.random.default_rng(0)
    for _ in range(20):
        n, batch, block = 60, 8, 4
        stack, top = ref.free_stack_init(n, rng.permutation(n).astype(np.int32))
        refs, bt, lens = np.zeros(n, np.int32), np.full((batch, 12), -1, np.int32), np.zeros(batch, np.int32)
        pool = torch.zeros(n, 2)
        for _ in range(30):
            what = rng.integers(4)
            if what == 0:
                new = rng.integers(0, 6, batch) * (lens < 40)
                if rng.random() < 0.5:
                    new = new * (lens > 0)
                _, top = ref.reserve(stack, top, bt, lens, new, block)
            elif what == 1 and (lens > 0).any() and (lens == 0).any():
                src, dst = rng.choice(np.flatnonzero(lens > 0)), rng.choice(np.flatnonzero(lens == 0))
                if top > 0:
                    top = ora.fork(stack, top, refs, bt, lens, [src], [dst], block, [pool])
            elif what == 2:
                top = ora.release(stack, top, refs, bt, lens, (rng.random(batch) < 0.3) & (lens > 0), block)
            else:
                stack, top, _ = ora.compact([pool], refs, bt, lens, block)
            ora.check(refs, stack, top, bt, lens, block)
