"""Compactions of more 4 KB slices than one copy launch counts, and of tables of many entries."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _books(dev, n_pages, width, lens, block, shared, seed):
    """A table of random pages of which some are held twice, and everything that a compaction takes."""
    rng = np.random.default_rng(seed)
    need = int(sum(-(-n // block) for n in lens))
    pages = np.sort(rng.choice(n_pages, need, replace=False))[rng.permutation(need)].astype(np.int32)
    bt, at = np.full((len(lens), width), -1, np.int32), 0
    refs = np.zeros(n_pages, np.int32)
    for b, n in enumerate(lens):
        p = -(-n // block)
        bt[b, :p] = pages[at:at + p]
        at += p
    if shared and n >= block:  # the last sequence holds the first one's whole pages
        k = min(lens[0], lens[-1]) // block
        bt[-1, :k] = bt[0, :k]
        refs[bt[0, :k]] = 1
    i32 = dict(dtype=torch.int32, device=dev)
    d = dict(bt=torch.as_tensor(bt, device=dev), lens=torch.tensor(lens, **i32), refs=torch.as_tensor(refs, device=dev),
             stack=torch.zeros(n_pages, **i32), top=torch.zeros(1, **i32), ws=torch.zeros(3 * n_pages, **i32),
             info=torch.zeros(2, **i32))
    return bt, refs, d


def _compact_and_check(dev, pools, bt, refs, d, lens, block, shared):
    from saint_kv import ops

    n_pages = pools[0].shape[0]
    held = np.unique(bt[bt >= 0])
    ids = torch.as_tensor(held, device=dev).long()
    g = torch.Generator(device=dev).manual_seed(1)
    before = []
    for p in pools:
        p[ids] = torch.randint(0, 256, (len(held), *p.shape[1:]), generator=g, device=dev, dtype=torch.uint8)
        before.append(p[ids])
    ops.compact(pools, d["bt"], d["lens"], block, d["stack"], d["top"], d["ws"], d["info"],
                refs=d["refs"] if shared else None)
    live = len(held)
    movers, holes = held[held >= live], np.setdiff1d(np.arange(live), held)
    assert d["info"].tolist() == [live, len(movers)] and int(d["top"]) == n_pages - live and len(movers) > 0
    new = np.arange(n_pages)
    new[movers] = holes
    want = np.where(bt >= 0, new[np.maximum(bt, 0)], -1)
    assert np.array_equal(d["bt"].cpu().numpy(), want)
    to = torch.as_tensor(new[held], device=dev).long()
    for p, b in zip(pools, before):
        assert torch.equal(p[to], b)
    stack = d["stack"][:n_pages - live].cpu().numpy()
    assert np.array_equal(stack[::-1], np.arange(live, n_pages))
    assert not d["ws"][:n_pages].any()
    if shared:
        moved = refs.copy()
        moved[holes], moved[movers] = refs[movers], 0
        assert np.array_equal(d["refs"].cpu().numpy(), moved)


@pytest.mark.parametrize("shared", [True, False])
def test_many_pools_of_many_pages(dev, shared) -> None:
    """Sixteen pools, together more slices than a launch counts."""
    n_pages, block, lens = (1 << 20) + 77, 16, [16 * 40, 5, 16 * 3000 + 1, 0, 16 * 40]
    bt, refs, d = _books(dev, n_pages, 3001, lens, block, shared, seed=0)
    pools = [torch.empty(n_pages, block, 34, dtype=torch.uint8, device=dev) for _ in range(16)]
    _compact_and_check(dev, pools, bt, refs, d, lens, block, shared)


def test_pages_of_several_launches(dev) -> None:
    """A page whose slices do not fit one launch for so many pages."""
    n_pages, block, lens = 1 << 23, 16, [16 * 500, 33, 16 * 2000 + 1]
    bt, refs, d = _books(dev, n_pages, 2001, lens, block, True, seed=1)
    pools = [torch.empty(n_pages, block, 1, 272, dtype=torch.uint8, device=dev)]  # two slices
    _compact_and_check(dev, pools, bt, refs, d, lens, block, True)


def test_tables_of_many_entries(dev) -> None:
    batch, width, block = 4096, 4097, 16
    lens = [0] * batch
    lens[7], lens[4000], lens[batch - 1] = 16 * 4097, 16 * 100 + 3, 16 * 4097
    for shared in (True, False):
        bt, refs, d = _books(dev, 20000, width, lens, block, False, seed=2)
        pools = [torch.empty(20000, block, 34, dtype=torch.uint8, device=dev)]
        _compact_and_check(dev, pools, bt, refs, d, lens, block, shared)
