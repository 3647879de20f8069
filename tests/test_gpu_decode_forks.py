"""Forks of a DecodeCache beside what callers do around them: graphs recorded before the first
fork, releases whose words are read later, attention before the next step, sequences named twice."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_fork import _decode_cache, _rows

pytestmark = pytest.mark.gpu


def _state(cache):
    """Tables, counts and free lists."""
    got = [cache.tok_lens.clone()]
    for g in cache.groups:
        got += [g.block_table.clone(), g.n_entries.clone(), g.free_top.clone(), g.free_stack[:int(g.free_top)].clone()]
        got += [] if g.refs is None else [g.refs.clone()]
    return got


def _prefilled(dev, lens, **kw):
    cache = _decode_cache(dev, **kw)
    cache.prefill(np.array(lens), data=_rows(cache, torch.Generator(device=dev).manual_seed(0), 5, max(lens)))
    return cache


def _recorded(cache, mask):
    """A graph of the mask's release and of a compaction; the host's lengths stay (recording runs nothing)."""
    m_dev = torch.as_tensor(mask.astype(np.uint8), device=cache.device)
    lens, graph = cache.host_lens.copy(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.release(mask, m_dev, check=False)
        cache.compact(sync=False)
    cache.host_lens = lens
    return graph, m_dev


@pytest.mark.parametrize("what", ["release", "compact"])
def test_no_fork_after_calls_of_one_owner_were_recorded(dev, what) -> None:
    """A graph of a release or a compaction without counts would free or move shared pages: the fork is refused."""
    cache = _prefilled(dev, [203, 0, 77, 0, 20])
    mask = np.array([0, 0, 0, 0, 1], dtype=bool)
    m_dev = torch.as_tensor(mask.astype(np.uint8), device=dev)
    lens, graph = cache.host_lens.copy(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if what == "release":
            cache.release(mask, m_dev, check=False)
        else:
            cache.compact(sync=False)
    cache.host_lens = lens
    before = _state(cache)
    with pytest.raises(RuntimeError, match="forks=True"):
        cache.fork(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(_state(cache), before)) and cache.host_lens.tolist() == lens.tolist()
    graph.replay()  # as good as ever while no page is shared
    torch.cuda.synchronize()
    if what == "release":
        cache.host_lens[mask] = 0
        assert cache.tok_lens.tolist() == [203, 0, 77, 0, 0]
    cache.check_release()


def test_a_release_recorded_before_the_first_fork(dev) -> None:
    """With forks=True: replays after forks, compared with a cache that makes the same calls eagerly."""
    cache, eager = (_prefilled(dev, [203, 0, 77, 0, 20], forks=True) for _ in range(2))
    mask = np.array([1, 0, 0, 0, 1], dtype=bool)
    graph, _ = _recorded(cache, mask)
    for round_ in range(4):
        for c in (cache, eager):
            if round_ == 0:
                c.fork(0, 1)
            else:
                c.fork([1, 2], [0, 4])  # sequence 1 lives on
        graph.replay()
        cache.host_lens[mask] = 0
        eager.release(mask)
        eager.compact()
        torch.cuda.synchronize()
        cache.check_release()
        for a, b in zip(_state(cache), _state(eager)):
            assert torch.equal(a, b)
        for g, gi in zip(cache.groups, range(len(cache.groups))):
            live = g.n_pages - int(g.free_top)
            held = g.block_table[g.block_table >= 0]
            assert held.unique().numel() == live
            for x, y in zip(cache._group_pools(gi), eager._group_pools(gi)):
                assert torch.equal(x[:live], y[:live])
        for c in (cache, eager):
            c.step()
            c.check_status()
            c.release(np.array([1, 0, 0, 1, 1], dtype=bool))  # a step gives every slot a token


def test_counts_from_the_start_change_nothing_else(dev) -> None:
    plain, counted = _prefilled(dev, [203, 50, 77, 8, 1]), _prefilled(dev, [203, 50, 77, 8, 1], forks=True)
    for c in (plain, counted):
        c.release(np.array([0, 1, 0, 0, 1], dtype=bool))
        c.compact()
        c.step()
        c.check_status()
    assert all(g.refs is None for g in plain.groups) and not any(g.refs.any() for g in counted.groups)
    for a, b in zip(plain.groups, counted.groups):
        assert torch.equal(a.block_table, b.block_table) and torch.equal(a.n_entries, b.n_entries)
        top = int(a.free_top)
        assert top == int(b.free_top) and torch.equal(a.free_stack[:top], b.free_stack[:top])


def test_no_forks(dev) -> None:
    """Nothing named, nothing done: the decode cache, the 4-bit cache and the call below them."""
    from saint_kv import Fp4TokenCache, ops

    cache = _prefilled(dev, [203, 0, 77, 0, 20])
    before = _state(cache)
    cache.fork([], [])
    assert all(torch.equal(a, b) for a, b in zip(_state(cache), before))
    four = Fp4TokenCache(1, 2, 64, 1, 64, block_size=16, device=dev)
    four.reserve(20)
    four.fork([], [])
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    ops.fork(four.free_stack, four.free_top, four.refs, four.block_table, four.seq_lens, none, none, 16, four.pool,
             four.status)
    ops.copy_slots([four.seq_lens], none, none)
    assert four.seq_lens.tolist() == four.host_lens.tolist() == [20, 20] and four.host_free == int(four.free_top)


def test_a_source_that_is_a_destination_too(dev) -> None:
    """All copies are of what the sources were before the call: of an empty one, an empty sequence."""
    cache = _prefilled(dev, [203, 0, 77, 0, 0])
    cache.fork([0, 1, 3], [1, 3, 4])
    assert cache.host_lens.tolist() == cache.tok_lens.tolist() == [203, 203, 77, 0, 0]
    for g in cache.groups:
        assert g.n_entries.tolist() == [n // g.m for n in (203, 203, 77, 0, 0)]
    cache.fork([3], [4])
    assert cache.tok_lens.tolist() == [203, 203, 77, 0, 0]
    cache.release(np.array([1, 1, 1, 0, 0], dtype=bool))
    for g in cache.groups:
        assert int(g.free_top) == g.n_pages


def test_a_fork_keeps_the_word_of_a_release(dev) -> None:
    cache = _prefilled(dev, [203, 0, 77, 0, 20])
    g = cache.groups[0]
    top = g.free_top.clone()
    g.free_top.fill_(g.n_pages)  # the pages would not fit: refused
    cache.release(np.array([0, 0, 0, 0, 1], dtype=bool), check=False)
    g.free_top.copy_(top)
    cache.fork(0, 1)
    with pytest.raises(RuntimeError, match="release refused"):
        cache.check_release()


def test_a_refused_fork_is_no_refused_release(dev) -> None:
    cache = _prefilled(dev, [101, 110, 0, 0, 0], pages_per_group={4: 30, 8: 8})
    with pytest.raises(RuntimeError, match="fork refused"):
        cache.fork([1, 1], [2, 3])
    cache.check_release()
    cache.release(np.array([1, 0, 0, 0, 0], dtype=bool))


def test_attention_of_a_fork_before_the_next_step(dev) -> None:
    """The last step's picks are the source's."""
    from saint_kv import DecodeCache, LayerSpec

    layers = [LayerSpec("csa", m=4, top_k=32), LayerSpec("hca", m=128), LayerSpec("swa")]
    cache = DecodeCache(layers, 3, 2048, window=32, block_size=16, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)
    cache.prefill(np.array([1500, 300, 0]), generator=g)
    for i in range(3):
        for x in cache.inputs[i].values():
            x.normal_(generator=g)
    cache.scores[0].normal_(generator=g)
    cache.step()
    cache.check_status()
    q = torch.randn(3, 16, cache.latent, generator=g, device=dev).to(torch.bfloat16)
    knw = torch.ones(cache.latent, device=dev)
    want = [cache.attention(i, q, None if layers[i].kind == "swa" else knw).clone() for i in range(3)]
    cache.release(np.array([0, 1, 1], dtype=bool))
    cache.fork([0, 0], [1, 2])
    q[1] = q[2] = q[0]
    for i in range(3):
        got = cache.attention(i, q, None if layers[i].kind == "swa" else knw)
        for b in range(3):
            assert torch.equal(got[b], got[0])
        assert torch.equal(got[0], want[i][0])
