"""Fp4TokenCache between a reservation and the next: forks, the tokens that are still to be
written, padded batches, and refusals that the device reports."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_fp4_cache import DIM, HEADS, KV, LAYERS, Model, new_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[37, 20, 0, 0, 5], [1, 1, 0, 0, 1], [16, 32, 0, 0, 3]])
def test_attention_right_after_a_fork(dev, counts) -> None:
    """A fork of a ragged prompt gives its source's outputs, and the others give what they gave."""
    cache = new_cache(dev)
    m = Model(dev, cache)
    want = m.step(np.array(counts))
    cache.fork([0, 1], [3, 2])
    m.q[3], m.q[2] = m.q[0], m.q[1]
    got = cache.attention(LAYERS - 1, m.q)
    for b in (0, 1, 4):
        assert torch.equal(got[b], want[-1][b])
    assert torch.equal(got[3], got[0]) and torch.equal(got[2], got[1])
    # a sequence that left and whose place another takes
    cache.release(np.array([0, 0, 0, 0, 1]))
    cache.fork([1], [4])
    m.q[4] = m.q[1]
    got = cache.attention(LAYERS - 1, m.q)
    assert torch.equal(got[4], got[1]) and torch.equal(got[0], want[-1][0])
