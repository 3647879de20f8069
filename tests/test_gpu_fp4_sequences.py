"""Fp4TokenCache between a reservation and the next: forks, the tokens that are still to be
written, padded batches, and refusals that the device reports."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_fp4_cache import DIM, HEADS, KV, LAYERS, Model, new_cache

pytestmark = pytest.mark.gpu


def _books(cache):
    return [x.clone() for x in (cache.block_table, cache.seq_lens, cache.refs, cache.free_top, cache.free_stack)]


def _same(cache, before, lens) -> None:
    assert all(torch.equal(a, b) for a, b in zip(_books(cache), before))
    assert cache.host_lens.tolist() == list(lens) and cache.host_free == int(cache.free_top)


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


def _rows(dev, t, heads=KV):
    return torch.ones(5, t, heads, DIM, dtype=torch.bfloat16, device=dev)


def test_a_fork_of_tokens_to_be_written_is_refused(dev) -> None:
    """Until every layer has them; forks of the other sequences go on, and the tokens still can be written."""
    cache = new_cache(dev)
    Model(dev, cache).step(np.array([20, 18, 0, 0, 0]))
    cache.reserve(np.array([16, 0, 0, 0, 0]))
    before = _books(cache)
    for i in range(LAYERS):
        with pytest.raises(RuntimeError, match="not been appended"):
            cache.fork([1, 0], [2, 3])
        _same(cache, before, [36, 18, 0, 0, 0])
        if i == 1:
            cache.fork([1], [2])
            before = _books(cache)
            cache.release(np.array([0, 0, 1, 0, 0]))
            before = _books(cache)
        cache.append(i, _rows(dev, 16), _rows(dev, 16))
    cache.fork([1, 0], [2, 3])
    assert cache.host_lens.tolist() == [36, 18, 18, 36, 0]


def test_an_append_after_a_fork_needs_a_reservation(dev) -> None:
    """The tokens reserved last lie in pages that are shared now."""
    cache = new_cache(dev)
    Model(dev, cache).step(np.array([32, 0, 0, 0, 0]))
    cache.fork([0], [1])
    before = [p.clone() for p in cache.pool]
    with pytest.raises(RuntimeError, match="reserve"):
        cache.append(0, _rows(dev, 32), _rows(dev, 32))
    assert all(torch.equal(a, b) for a, b in zip(cache.pool, before))
    Model(dev, cache).step(np.array([1, 1, 0, 0, 0]))


def test_appends_that_a_graph_replays(dev) -> None:
    """Steps of an eager reservation and a replayed append and attention, with forks between them."""
    cache, eager = new_cache(dev), new_cache(dev)
    for c in (cache, eager):
        Model(dev, c).step(np.array([20, 33, 0, 0, 0]))
    g = torch.Generator(device=dev).manual_seed(3)
    k, v, q = (torch.randn(5, 1, h, DIM, generator=g, device=dev).to(torch.bfloat16) for h in (KV, KV, HEADS))

    def layers(c):
        for i in range(LAYERS):
            c.append(i, k, v)
        return [c.attention(i, q) for i in range(LAYERS)]

    for c in (cache, eager):
        c.reserve(1)
        layers(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layers(cache)
    for n in range(3):
        for c in (cache, eager):
            c.release(np.array([0, 0, 1, 1, 0]))
            c.fork([1, 0], [2, 3])
            c.reserve(1)
        for x in (k, v, q):
            x.normal_(generator=g)
        graph.replay()
        want = layers(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n


def test_a_refusal_is_reported_whatever_comes_after(dev) -> None:
    """The device refuses where the free list was changed behind the host's back; later calls succeed."""
    cache = new_cache(dev)
    Model(dev, cache).step(np.array([20, 0, 0, 0, 0]))

    def without_pages(call):
        top = cache.free_top.clone()
        cache.free_top.zero_()
        call()
        cache.free_top.copy_(top)

    for later in (1, 200):
        for refused in (lambda: cache.reserve(np.array([0, 17, 0, 0, 0])), lambda: cache.fork([0], [2])):
            without_pages(refused)
            for _ in range(later):
                cache.reserve(0)
            with pytest.raises(RuntimeError, match="refused"):
                cache.check_status()
            assert cache.host_lens.tolist() == cache.seq_lens.tolist() == [20, 0, 0, 0, 0]
            assert cache.host_free == int(cache.free_top)
            cache.check_status()  # reported once
    without_pages(lambda: cache.reserve(np.array([0, 17, 0, 0, 0])))
    cache.reserve(0)
    with pytest.raises(RuntimeError, match="refused"):
        cache.release(np.array([1, 0, 0, 0, 0]))
    assert cache.host_lens.tolist() == cache.seq_lens.tolist() and cache.host_free == int(cache.free_top)


def test_scales_that_fp32_takes_for_zero_are_refused(dev) -> None:
    """Zero stands for the default scale and for no cap in the descriptor."""
    from saint_kv import fp4_attention

    cache = new_cache(dev)
    Model(dev, cache).step(1)
    q = _rows(dev, 1, HEADS)
    for kw in (dict(scale=1e-50), dict(softcap=1e-50), dict(scale=1e-50, softcap=2.0)):
        with pytest.raises(ValueError, match="fp32"):
            fp4_attention(q, cache.pool[0], cache.block_table, cache.seq_lens, **kw)
        with pytest.raises(ValueError, match="fp32"):
            cache.attention(0, q, **kw)


def test_tokens_that_do_not_fit_the_reservation(dev) -> None:
    """Queries or rows of more or fewer tokens than were reserved, where nothing says which they are."""
    cache = new_cache(dev)
    cache.reserve(5)
    with pytest.raises(ValueError, match="5"):
        cache.append(0, _rows(dev, 4), _rows(dev, 4))
    cache.append(0, _rows(dev, 8), _rows(dev, 8))  # a padded batch: the first five
    with pytest.raises(ValueError, match="5"):
        cache.attention(0, _rows(dev, 8, HEADS))
    cache.attention(0, _rows(dev, 5, HEADS))
    cache.attention(0, _rows(dev, 1, HEADS))  # the newest
    cache.reserve(np.array([5, 3, 0, 1, 1]))
    with pytest.raises(ValueError, match="5"):
        cache.append(0, _rows(dev, 4), _rows(dev, 4))
    cache.append(0, _rows(dev, 8), _rows(dev, 8))
    cache.attention(0, _rows(dev, 8, HEADS))
    for _ in range(2):  # the newest of two reservations
        cache.reserve(2)
        cache.append(0, _rows(dev, 2), _rows(dev, 2))
    cache.attention(0, _rows(dev, 4, HEADS))


def test_rows_for_more_tokens_than_a_sequence_has(dev) -> None:
    """One expanded token as the rows of 2^28, of which a few are new: as many as a launch's grid cannot count."""
    from saint_kv import ops

    pool = ops.fp4_pool(4, 16, 1, 512, dev)
    i32 = dict(dtype=torch.int32, device=dev)
    bt, lens = torch.tensor([[2, 0], [3, 1]], **i32), torch.tensor([20, 3], **i32)
    k, v = (torch.randn(2, 1, 1, 512, device=dev).to(torch.bfloat16) for _ in range(2))
    ops.fp4_quant_append(pool, bt, lens, k.expand(2, 1 << 28, 1, 512), v.expand(2, 1 << 28, 1, 512), lens)
    want = ops.fp4_pool(4, 16, 1, 512, dev)
    ops.fp4_quant_append(want, bt, lens, k.expand(2, 20, 1, 512), v.expand(2, 20, 1, 512), lens)
    assert torch.equal(pool, want)


def test_slots_of_nothing(dev) -> None:
    """Arrays without bytes, or without slots, beside others."""
    from saint_kv import ops

    idx = torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device=dev)
    full = torch.arange(12, device=dev).view(4, 3)
    ops.copy_slots([torch.zeros(4, 0, device=dev), full, torch.zeros(4, 2, 0, device=dev)], idx[0], idx[1])
    assert full.tolist() == [[0, 1, 2], [0, 1, 2], [6, 7, 8], [6, 7, 8]]
    ops.copy_slots([torch.zeros(4, 0, device=dev)], idx[0], idx[1])
    ops.copy_slots([torch.zeros(0, 3, device=dev)], idx[0], idx[1])


def test_a_cache_on_another_device_than_the_current_one(dev, monkeypatch) -> None:
    """Every launch finds the cache's device current, and the caller's is current again behind it."""
    from saint_kv import Fp4TokenCache, _lib

    here, call, seen = [1], _lib.call, []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: here[0])
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: here.__setitem__(0, i))
    monkeypatch.setattr(_lib, "call", lambda name, *args: (seen.append((name, here[0])), call(name, *args))[1])
    cache = Fp4TokenCache(LAYERS, 5, 160, KV, DIM, block_size=16, device=dev)
    cache.reserve(np.array([37, 0, 5, 1, 0]))
    for i in range(LAYERS):
        cache.append(i, _rows(dev, 37), _rows(dev, 37))
        cache.attention(i, _rows(dev, 37, HEADS))
    cache.fork([0], [1])
    cache.release(np.array([1, 0, 0, 0, 0]))
    cache.compact()
    assert here == [1] and {d for _, d in seen} == {0}
    assert {n for n, _ in seen} == {"skv_free_stack_init", "skv_reserve", "skv_fp4_quant_append", "skv_fp4_attention",
                                    "skv_fork", "skv_copy_slots", "skv_release_shared", "skv_compact_shared"}
