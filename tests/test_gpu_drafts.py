"""Drafted trees on the GPU against the plain oracle: masks and depths, accepted paths, kept tokens, and the whole step of a
cache that drafts, checks and keeps.  Everything here is whole numbers or bytes: equal, or wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_fp4_view import check

from oracle import drafts
from oracle import fp4_cache as ora
from oracle import shared_pages

pytestmark = pytest.mark.gpu


def trees(rng, batch: int, t: int, chain: float = 0.6, bad: float = 0.0) -> np.ndarray:
    parents = np.full((batch, t), -1, dtype=np.int32)
    for b in range(batch):
        for i in range(1, t):
            parents[b, i] = i - 1 if rng.random() < chain else rng.integers(0, i)
            if rng.random() < bad:
                parents[b, i] = rng.choice([-1, -2, i, i + 1, t, 1 << 30, -(1 << 31)])
    return parents


@pytest.mark.parametrize("batch,t", [(1, 1), (3, 2), (2, 63), (5, 64), (4, 65), (2, 128), (2, 300), (1, 1024)])
@pytest.mark.parametrize("bad", [0.0, 0.05])
def test_masks_and_depths(dev, batch, t, bad) -> None:
    from saint_kv import ops

    rng = np.random.default_rng(t)
    parents = trees(rng, batch, t, chain=0.9 if t > 200 else 0.5, bad=bad)
    counts = rng.integers(-2, t + 3, batch).astype(np.int32)
    for n_new in (None, counts):
        n = np.full(batch, t) if n_new is None else np.clip(n_new, 0, t)
        seen = ora.tree_masks(parents, n)
        tree, depths = ops.draft_tree(torch.as_tensor(parents, device=dev),
                                      None if n_new is None else torch.as_tensor(n_new, device=dev))
        assert np.array_equal(tree.cpu().numpy(), ora.pack_masks(seen))
        assert np.array_equal(depths.cpu().numpy(), np.maximum(seen.sum(-1) - 1, 0))


@pytest.mark.parametrize("batch,t", [(1, 1), (3, 2), (2, 63), (5, 64), (4, 65), (2, 128), (2, 300), (1, 1024)])
@pytest.mark.parametrize("wide", [False, True])
def test_accepted_paths(dev, batch, t, wide) -> None:
    """Few names for the tokens, so that paths are long and siblings share them."""
    from saint_kv import ops

    rng = np.random.default_rng(t + wide)
    parents = trees(rng, batch, t, chain=0.7, bad=0.02)
    kind = np.int64 if wide else np.int32
    tokens = rng.integers(0, 3, (batch, t)).astype(kind)
    picks = np.where(rng.random((batch, t)) < 0.1, -1, rng.integers(0, 2, (batch, t))).astype(kind)
    if wide:  # ids past 32 bits are told apart
        tokens[:, 1::2] += 1 << 32
    counts = rng.integers(-1, t + 2, batch).astype(np.int32)
    for n_new in (None, counts):
        want = drafts.accept(parents, tokens, picks, np.full(batch, t) if n_new is None else n_new)
        # one pick a row of a wider table, as the most likely tokens come
        table = torch.zeros(batch, t, 5, dtype=torch.int64 if wide else torch.int32, device=dev)
        table[..., 0] = torch.as_tensor(picks, device=dev)
        got = ops.accept_drafts(torch.as_tensor(parents, device=dev), torch.as_tensor(tokens, device=dev), table[..., 0],
                                None if n_new is None else torch.as_tensor(n_new, device=dev))
        for g, w in zip(got, want):
            assert g.dtype == torch.from_numpy(w).dtype and np.array_equal(g.cpu().numpy(), w)


def filled(dev, rng, lens, block, heads, dim, layers, spare=3, extra=2):
    """Pools of random bytes, a shuffled table, a free stack with room for every page."""
    lens = np.asarray(lens, dtype=np.int32)
    pages = -(-lens // block)
    n_pages = int(pages.sum()) + spare
    order = rng.permutation(n_pages).astype(np.int32)
    bt = np.full((len(lens), max(1, int(pages.max(initial=0))) + extra), -1, dtype=np.int32)
    at = 0
    for b, p in enumerate(pages):
        bt[b, :p] = order[at:at + p]
        at += p
    stack = np.zeros(n_pages, dtype=np.int32)
    stack[:n_pages - at] = order[at:]
    pools = [rng.integers(0, 256, (n_pages, block, heads, dim * 17 // 16), dtype=np.uint8) for _ in range(layers)]
    return pools, bt, lens, stack, n_pages - at


def paths(rng, n_new, width):
    path, n_keep = np.full((len(n_new), width), -1, dtype=np.int32), np.zeros(len(n_new), dtype=np.int32)
    for b, n in enumerate(n_new):
        k = int(rng.integers(0, min(int(n), width) + 1))
        path[b, :k] = np.sort(rng.choice(int(n), k, replace=False))
        n_keep[b] = k
    return path, n_keep


def run_keep(dev, pools, bt, lens, stack, top, n_new, path, n_keep, refs=None, **kw):
    from saint_kv import ops

    def gpu(x):
        return torch.as_tensor(x.copy(), device=dev)

    p, state = [gpu(x) for x in pools], [gpu(x) for x in (stack, np.array([top], dtype=np.int32), bt, lens)]
    status = torch.full((1,), 77, dtype=torch.int32, device=dev)
    n = n_new if isinstance(n_new, int) else gpu(np.asarray(n_new, dtype=np.int32))
    ops.keep_tokens(*state, n, gpu(np.asarray(path, dtype=np.int32)), gpu(np.asarray(n_keep, dtype=np.int32)), p, status,
                    refs=None if refs is None else gpu(refs), **kw)
    return [x.cpu().numpy() for x in p], [x.cpu().numpy() for x in state], int(status.item())


SHAPES = [
    # batch, longest, newest, path's width, block, heads, dim, layers
    (1, 40, 8, 8, 16, 1, 32, 1), (3, 100, 33, 33, 16, 3, 96, 2), (5, 200, 64, 64, 32, 2, 128, 3), (2, 300, 200, 256, 16, 1, 512, 1),
    (7, 90, 12, 12, 64, 8, 64, 16), (4, 70, 20, 9, 48, 2, 160, 2), (2, 2000, 1024, 1024, 128, 1, 224, 1), (70, 50, 17, 17, 16, 1, 64, 1),
]


@pytest.mark.parametrize("batch,longest,newest,width,block,heads,dim,layers", SHAPES)
def test_kept_tokens(dev, batch, longest, newest, width, block, heads, dim, layers) -> None:
    rng = np.random.default_rng(batch + dim)
    lens = rng.integers(0, longest + 1, batch)
    n_new = np.minimum(rng.integers(0, newest + 1, batch), lens)
    pools, bt, lens, stack, top = filled(dev, rng, lens, block, heads, dim, layers)
    path, n_keep = paths(rng, n_new, width)
    got, books, status = run_keep(dev, pools, bt, lens, stack, top, n_new, path, n_keep)
    want = [x.copy() for x in pools]
    top, ok = drafts.keep(stack, top, bt, lens, n_new, path, n_keep, want)
    assert (status, ok) == (0, 0)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    assert int(books[1][0]) == top and np.array_equal(books[0][:top], stack[:top])
    assert np.array_equal(books[2], bt) and np.array_equal(books[3], lens)


def test_one_count_for_all(dev) -> None:
    rng = np.random.default_rng(3)
    pools, bt, lens, stack, top = filled(dev, rng, [50, 33, 64], 16, 2, 64, 2)
    path, n_keep = paths(rng, [20, 20, 20], 20)
    n_keep[1], path[1] = 0, -1  # all of them dropped
    got, books, status = run_keep(dev, pools, bt, lens, stack, top, 20, path, n_keep)
    top, _ = drafts.keep(stack, top, bt, lens, np.full(3, 20), path, n_keep, pools)
    assert status == 0 and all(np.array_equal(g, w) for g, w in zip(got, pools))
    assert int(books[1][0]) == top and np.array_equal(books[2], bt) and np.array_equal(books[3], lens)


def test_refused_keeps_write_nothing(dev) -> None:
    rng = np.random.default_rng(5)
    pools, bt, lens, stack, top = filled(dev, rng, [50, 33, 64], 16, 2, 64, 2)
    n_new, path, n_keep = [20, 9, 33], np.full((3, 33), -1, dtype=np.int32), np.array([3, 2, 4], dtype=np.int32)
    path[0, :3], path[1, :2], path[2, :4] = [0, 4, 7], [1, 8], [0, 1, 2, 9]
    refs = np.zeros(len(stack), dtype=np.int32)

    def variant(**over):
        a = dict(pools=pools, bt=bt.copy(), lens=lens.copy(), stack=stack, top=top, n_new=list(n_new), path=path.copy(),
                 n_keep=n_keep.copy(), refs=refs.copy())
        for k, v in over.items():
            if callable(v):
                v(a[k])
            else:
                a[k] = v
        return a

    def at(i, value):
        def go(x):
            x[i] = value
        return go

    cases = [variant(n_keep=at(1, 10)), variant(n_keep=at(0, -1)), variant(path=at((0, 2), 4)), variant(path=at((0, 2), 20)),
             variant(path=at((1, 0), -1)), variant(path=at((2, 3), 1)), variant(n_new=at(1, 34)), variant(n_new=at(1, -1)),
             variant(lens=at(0, -3)), variant(lens=at(0, 16 * bt.shape[1] + 1)), variant(bt=at((0, 2), -1)),
             variant(bt=at((2, 3), len(stack))), variant(top=-1), variant(top=len(stack) + 1),
             variant(refs=at(int(bt[0, 1]), 1)), variant(refs=at(int(bt[2, 3]), 2)), variant(top=len(stack) - 1)]
    for c in cases:
        got, books, status = run_keep(dev, **c)
        state = [c["stack"].copy(), c["bt"].copy(), c["lens"].copy()]
        _, want = drafts.keep(state[0], c["top"], state[1], state[2], np.array(c["n_new"]), c["path"], c["n_keep"],
                              [p.copy() for p in pools], c["refs"])
        assert want != 0 and status == want
        assert all(np.array_equal(g, w) for g, w in zip(got, pools))
        for g, w in zip(books, (c["stack"], [c["top"]], c["bt"], c["lens"])):
            assert np.array_equal(g, w)
    got, books, status = run_keep(dev, **variant())
    assert status == 0
    got, books, status = run_keep(dev, **variant(refs=at(int(bt[0, 0]), 1)))  # a whole page before is shared
    assert status == 0


def test_refusals_on_the_host(dev) -> None:
    from saint_kv import ops

    i32 = dict(dtype=torch.int32, device=dev)
    parents = torch.zeros(2, 8, **i32)
    for bad in (parents.long(), parents[0], torch.zeros(2, 0, **i32), torch.zeros(1, 1025, **i32), parents[:, ::2]):
        with pytest.raises(ValueError):
            ops.draft_tree(bad)
        with pytest.raises(ValueError):
            ops.accept_drafts(bad, parents, parents)
    with pytest.raises(ValueError):
        ops.draft_tree(parents, torch.zeros(3, **i32))
    with pytest.raises(RuntimeError, match="CPU"):
        ops.draft_tree(parents.cpu())
    for bad in (parents.short(), parents[:1], parents[:, :7]):
        with pytest.raises(ValueError):
            ops.accept_drafts(parents, bad, parents)
        with pytest.raises(ValueError):
            ops.accept_drafts(parents, parents, bad)
    pool, stack, top = ops.fp4_pool(4, 16, 1, 32, dev), torch.zeros(4, **i32), torch.zeros(1, **i32)
    bt, lens, n = torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(2, **i32)
    ok = dict(free_stack=stack, free_top=top, block_table=bt, seq_lens=lens, n_new=0, path=parents, n_keep=n, pools=[pool],
              status=torch.zeros(1, **i32))
    ops.keep_tokens(**ok)
    for bad in (dict(pools=[]), dict(pools=[pool] * 33), dict(pools=[pool, pool]), dict(pools=[pool, pool[:3]]), dict(pools=[pool.int()]), dict(n_new=-1),
                dict(free_stack=torch.zeros(5, **i32)), dict(path=parents[:1]), dict(path=torch.zeros(2, 0, **i32)),
                dict(path=torch.zeros(2, 1025, **i32)), dict(n_keep=n.long()), dict(refs=torch.zeros(3, **i32)),
                dict(workspace=torch.zeros(15, dtype=torch.uint8, device=dev)), dict(seq_lens=lens[:1])):
        with pytest.raises(ValueError):
            ops.keep_tokens(**{**ok, **bad})


def test_captured_steps_replay(dev) -> None:
    """Masks, paths and kept tokens in a graph, replayed with eager work between, each time as the eager calls do."""
    from saint_kv import ops

    rng = np.random.default_rng(1)
    pools, bt, lens, stack, top = filled(dev, rng, [70, 40, 33], 16, 2, 64, 2)
    t = 20
    i32 = dict(dtype=torch.int32, device=dev)
    books0 = [torch.as_tensor(x, device=dev) for x in (stack, np.array([top], dtype=np.int32), bt, lens)]
    p0 = [torch.as_tensor(x, device=dev) for x in pools]
    parents, tokens, picks = (torch.zeros(3, t, **i32) for _ in range(3))
    n_new = torch.zeros(3, **i32)

    def step(books, p, status):
        tree, depths = ops.draft_tree(parents, n_new)
        path, n_keep, following = ops.accept_drafts(parents, tokens, picks, n_new)
        ops.keep_tokens(*books, n_new, path, n_keep, p, status)
        return [tree, depths, path, n_keep, following]

    books, p, status = [x.clone() for x in books0], [x.clone() for x in p0], torch.zeros(1, **i32)
    step(books, p, status)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(books, p, status)
    for k in range(4):
        parents.copy_(torch.as_tensor(trees(rng, 3, t)))
        tokens.copy_(torch.as_tensor(rng.integers(0, 2, (3, t))))
        picks.copy_(torch.as_tensor(rng.integers(0, 2, (3, t))))
        n_new.copy_(torch.as_tensor(rng.integers(1, t + 1, 3)))
        for x, y in zip(books + p, books0 + p0):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        eager, ep, es = [x.clone() for x in books0], [x.clone() for x in p0], torch.zeros(1, **i32)
        want = step(eager, ep, es)
        assert int(status.item()) == 0
        for x, y in zip(outs + books + p, want + eager + ep):
            assert torch.equal(x, y)


def rows_of(dev, rng, *shape):
    return torch.as_tensor(rng.standard_normal(shape), dtype=torch.float32, device=dev).to(torch.bfloat16)


def test_a_drafting_cache_is_as_one_that_appends_what_was_accepted(dev) -> None:
    """Steps of reserve, append, attention, accept and keep over three layers against a cache that is given the accepted
    tokens alone: lengths, free pages, every byte of the tokens, and the attention of each accepted node."""
    from saint_kv import Fp4TokenCache, ops

    rng = np.random.default_rng(2)
    batch, heads, kv, dim, t, layers = 4, 8, 2, 128, 12, 3
    caches = [Fp4TokenCache(layers, batch, 400, kv, dim, block_size=16, device=dev) for _ in range(2)]
    prompt = np.array([40, 3, 0, 64])
    for cache in caches:
        cache.reserve(prompt)
    for i in range(layers):
        k, v = rows_of(dev, rng, batch, 64, kv, dim), rows_of(dev, rng, batch, 64, kv, dim)
        for cache in caches:
            cache.append(i, k, v)
    drafting, plain = caches
    for step in range(6):
        n_new = rng.integers(0 if step else 1, t + 1, batch)
        parents = trees(rng, batch, t)
        tokens, picks = rng.integers(0, 2, (batch, t)).astype(np.int32), rng.integers(0, 2, (batch, t)).astype(np.int32)
        n_gpu, p_gpu = torch.as_tensor(n_new.astype(np.int32), device=dev), torch.as_tensor(parents, device=dev)
        tree, _ = ops.draft_tree(p_gpu, n_gpu)
        path, n_keep, _ = ops.accept_drafts(p_gpu, torch.as_tensor(tokens, device=dev), torch.as_tensor(picks, device=dev), n_gpu)
        want_path, want_keep, _ = drafts.accept(parents, tokens, picks, n_new)
        assert np.array_equal(path.cpu().numpy(), want_path)
        drafting.reserve(n_new)
        plain.reserve(want_keep)
        for i in range(layers):
            k, v, q = rows_of(dev, rng, batch, t, kv, dim), rows_of(dev, rng, batch, t, kv, dim), rows_of(dev, rng, batch, t, heads, dim)
            drafting.append(i, k, v)
            out = drafting.attention(i, q, tree=tree)
            check(out, q, drafting.pool[i], drafting.block_table, drafting.seq_lens, seen=ora.tree_masks(parents, n_new),
                  n_new=n_new)
            at = path.long().clamp_min(0)
            kept = [x.gather(1, at[..., None, None].expand(-1, -1, *x.shape[2:])) for x in (k, v, q, out)]
            plain.append(i, kept[0], kept[1])
            seen = kept[3].masked_fill((path < 0)[..., None, None], 0)  # past the path: none
            check(seen, kept[2], plain.pool[i], plain.block_table, plain.seq_lens, n_new=want_keep)
        assert np.array_equal(drafting.keep(path, n_keep), want_keep)
        assert np.array_equal(drafting.host_lens, plain.host_lens) and drafting.host_free == plain.host_free
        assert torch.equal(drafting.seq_lens, plain.seq_lens) and int(drafting.free_top.item()) == drafting.host_free
        longest = int(plain.host_lens.max())
        for i in range(layers):
            got = []
            for cache in caches:
                o = [torch.zeros(batch, longest, kv, dim, dtype=torch.bfloat16, device=dev) for _ in range(2)]
                ops.fp4_gather(cache.pool[i], cache.block_table, cache.seq_lens, *o, cache.seq_lens)
                got.append(o)
            assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
        if step == 3:  # a sequence ends, and begins anew
            mask = np.array([True, False, False, True]) & (plain.host_lens > 0)
            for cache in caches:
                cache.release(mask)
    shared_pages.check(drafting.refs.cpu().numpy(), drafting.free_stack.cpu().numpy(), drafting.host_free,
                       drafting.block_table.cpu().numpy(), drafting.seq_lens.cpu().numpy(), 16)


def test_keeps_of_a_cache_that_forks(dev) -> None:
    from saint_kv import Fp4TokenCache, ops

    rng = np.random.default_rng(4)
    cache = Fp4TokenCache(1, 3, 200, 1, 64, block_size=16, device=dev)

    def append(n):
        cache.reserve(n)
        t = max(int(np.max(n)), 1)
        cache.append(0, rows_of(dev, rng, 3, t, 1, 64), rows_of(dev, rng, 3, t, 1, 64))

    def keep(lists):
        path = np.full((3, 40), -1, dtype=np.int32)
        for b, p in enumerate(lists):
            path[b, :len(p)] = p
        return cache.keep(torch.as_tensor(path, device=dev), torch.tensor([len(p) for p in lists], dtype=torch.int32, device=dev))

    append(np.array([35, 0, 0]))
    cache.fork([0], [1])
    with pytest.raises(RuntimeError, match="fork"):
        keep([[0], [0], []])
    append(np.array([20, 20, 0]))  # in pages of their own
    assert keep([[0, 5, 19], [], []]).tolist() == [3, 0, 0]
    assert cache.host_lens.tolist() == [38, 35, 0]
    cache.reserve(np.array([4, 4, 0]))
    with pytest.raises(RuntimeError, match="appended"):
        keep([[0], [0], []])
    cache.append(0, rows_of(dev, rng, 3, 4, 1, 64), rows_of(dev, rng, 3, 4, 1, 64))
    with pytest.raises(RuntimeError, match="refused"):
        keep([[0], [3, 2], []])
    assert cache.host_lens.tolist() == [42, 39, 0]
    assert keep([[0, 1, 2, 3], [2], []]).tolist() == [4, 1, 0]
    assert keep([[1], [0], []]).tolist() == [1, 1, 0]  # of those that stayed
    cache.release(np.array([True, False, False]))
    assert keep([[], [0], []]).tolist() == [0, 1, 0]  # a released sequence has none
    assert int(cache.free_top.item()) == cache.host_free
    shared_pages.check(cache.refs.cpu().numpy(), cache.free_stack.cpu().numpy(), cache.host_free,
                       cache.block_table.cpu().numpy(), cache.seq_lens.cpu().numpy(), 16)


def test_a_captured_keep_of_a_cache_is_refused(dev) -> None:
    """It reads back how many tokens stayed; nothing is recorded, and the cache is as it was."""
    from saint_kv import Fp4TokenCache

    cache = Fp4TokenCache(1, 1, 64, 1, 32, block_size=16, device=dev)
    cache.reserve(8)
    cache.append(0, torch.zeros(1, 8, 1, 32, dtype=torch.bfloat16, device=dev), torch.zeros(1, 8, 1, 32, dtype=torch.bfloat16, device=dev))
    path, n_keep = torch.zeros(1, 4, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="keep"):
            cache.keep(path, n_keep)
        path.zero_()
    graph.replay()
    assert cache.keep(path, n_keep).tolist() == [1] and cache.host_lens.tolist() == [1]


def test_mixed_ids_and_trees_on_another_stream(dev) -> None:
    """int32 tokens with int64 picks, on a stream of the caller's."""
    from saint_kv import ops

    rng = np.random.default_rng(9)
    parents, tokens, picks = trees(rng, 5, 40), rng.integers(0, 2, (5, 40)).astype(np.int32), rng.integers(0, 2, (5, 40))
    want = drafts.accept(parents, tokens, picks, np.full(5, 40))
    stream = torch.cuda.Stream(device=dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        got = ops.accept_drafts(*(torch.as_tensor(x, device=dev) for x in (parents, tokens, picks)))
        tree, _ = ops.draft_tree(torch.as_tensor(parents, device=dev))
    stream.synchronize()
    assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got, want)) and got[2].dtype == torch.int64
    assert np.array_equal(tree.cpu().numpy(), ora.pack_masks(ora.tree_masks(parents, np.full(5, 40))))


def test_far_pages(dev) -> None:
    """Pages whose bytes lie past 2^32."""
    from saint_kv import ops

    n_pages, block, heads, dim = 65000, 64, 8, 128
    pool = ops.fp4_pool(n_pages, block, heads, dim, dev)
    assert pool.numel() > 2 ** 32
    used = np.array([64999, 3, 64001, 62500], dtype=np.int64)
    at = torch.as_tensor(used, device=dev)
    rng = np.random.default_rng(8)
    small = rng.integers(0, 256, (4, block, heads, dim * 17 // 16), dtype=np.uint8)
    pool[at] = torch.as_tensor(small, device=dev)
    lens, n_new = np.array([130, 64], dtype=np.int32), np.array([90, 60], dtype=np.int32)
    path, n_keep = paths(rng, n_new, 90)
    where = np.array([[0, 1, 2], [3, -1, -1]], dtype=np.int32)
    bt = torch.as_tensor(np.where(where < 0, -1, used[where]).astype(np.int32), device=dev)
    stack, top = torch.zeros(n_pages, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    status, lens_t = torch.full((1,), 7, dtype=torch.int32, device=dev), torch.as_tensor(lens, device=dev)
    ops.keep_tokens(stack, top, bt, lens_t, torch.as_tensor(n_new, device=dev), torch.as_tensor(path, device=dev),
                    torch.as_tensor(n_keep, device=dev), [pool], status)
    free = np.zeros(4, dtype=np.int32)
    count, ok = drafts.keep(free, 0, where, lens, n_new, path, n_keep, [small])
    assert int(status.item()) == ok == 0 and int(top.item()) == count
    assert np.array_equal(pool[at].cpu().numpy(), small)
    assert np.array_equal(lens_t.cpu().numpy(), lens)
    assert np.array_equal(stack[:count].cpu().numpy(), used[free[:count]])
    assert np.array_equal(bt.cpu().numpy(), np.where(where < 0, -1, used[where]))


def test_an_earlier_refusal_leaves_what_stayed_in_order(dev) -> None:
    """It is raised by the keep, whose tokens have moved: the next keep counts from these; a keep's own refusal moves none."""
    from saint_kv import Fp4TokenCache

    cache = Fp4TokenCache(1, 2, 64, 1, 32, block_size=16, device=dev)
    rows = torch.randn(2, 9, 1, 32, generator=torch.Generator(device=dev).manual_seed(0), device=dev).to(torch.bfloat16)
    cache.reserve(9)
    cache.append(0, rows, rows)
    cache.status.fill_(4)  # as a launch before may have left it
    path = torch.tensor([[0, 2, 5, -1], [1, -1, -1, -1]], dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="refused"):
        cache.keep(path, torch.tensor([3, 1], dtype=torch.int32, device=dev))
    assert cache.host_lens.tolist() == [3, 1] == cache.seq_lens.tolist()
    with pytest.raises(RuntimeError, match="refused"):  # one of a sequence's single token twice
        cache.keep(path, torch.tensor([3, 2], dtype=torch.int32, device=dev))
    assert cache.host_lens.tolist() == [3, 1] == cache.seq_lens.tolist()
    path = torch.tensor([[1, 2], [0, -1]], dtype=torch.int32, device=dev)
    assert cache.keep(path, torch.tensor([2, 1], dtype=torch.int32, device=dev)).tolist() == [2, 1]
    assert cache.host_lens.tolist() == [2, 1] == cache.seq_lens.tolist()
    assert int(cache.free_top.item()) == cache.host_free


def books_of(cache):
    return [x.clone() for x in (cache.seq_lens, cache.block_table, cache.free_stack, cache.free_top, cache.refs, *cache.pool)]


@pytest.mark.parametrize("noticed", [False, True])
@pytest.mark.parametrize("counts", [30, np.array([30, 0, 20])])
def test_tokens_of_a_refused_reservation_are_not_kept(dev, counts, noticed) -> None:
    """The device refuses a reservation (its free pages were taken behind the host's back): a keep raises and leaves the
    committed tokens, also once the refusal has been raised, and after more status words than there are."""
    from saint_kv import Fp4TokenCache

    rng = np.random.default_rng(6)
    cache = Fp4TokenCache(2, 3, 256, 1, 32, block_size=16, device=dev)

    def append(n):
        cache.reserve(n)
        t = int(np.max(n))
        for i in range(2):
            cache.append(i, rows_of(dev, rng, 3, t, 1, 32), rows_of(dev, rng, 3, t, 1, 32))

    append(np.array([40, 35, 64]))
    path = torch.tensor([[0, 2, 5], [0, -1, -1], [1, 2, -1]], dtype=torch.int32, device=dev)
    n_keep = torch.tensor([3, 0, 2] if isinstance(counts, np.ndarray) else [3, 1, 2], dtype=torch.int32, device=dev)
    free = cache.free_top.clone()
    cache.free_top.zero_()
    append(counts)
    before = books_of(cache)
    if noticed:
        with pytest.raises(RuntimeError, match="refused"):
            cache.check_status()
    else:
        for _ in range(200):  # of other calls
            cache._status_word()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="refused"):
            cache.keep(path, n_keep)
        assert all(torch.equal(x, y) for x, y in zip(books_of(cache), before))
        assert cache.host_lens.tolist() == [40, 35, 64] and cache.host_free == 0
    # nothing of the refused one is left: none of its tokens can be kept or must be appended
    assert cache.keep(path, torch.zeros_like(n_keep)).tolist() == [0, 0, 0]
    assert all(torch.equal(x, y) for x, y in zip(books_of(cache), before))
    cache.free_top.copy_(free)
    cache.host_free = int(free.item())
    append(np.array([6, 3, 4]))
    assert cache.keep(path, n_keep).tolist() == n_keep.tolist()
    assert cache.host_lens.tolist() == (np.array([40, 35, 64]) + n_keep.cpu().numpy()).tolist() == cache.seq_lens.tolist()
    assert int(cache.free_top.item()) == cache.host_free


def test_a_reservation_after_a_refused_one_is_kept(dev) -> None:
    """An earlier refusal that nobody has read is raised; the tokens reserved since have moved, and count."""
    from saint_kv import Fp4TokenCache

    cache = Fp4TokenCache(1, 2, 256, 1, 32, block_size=16, device=dev)
    rows = rows_of(dev, np.random.default_rng(0), 2, 40, 1, 32)
    cache.reserve(40)
    cache.append(0, rows, rows)
    free = cache.free_top.clone()
    cache.free_top.zero_()
    cache.reserve(30)  # refused
    cache.free_top.copy_(free)
    cache.reserve(5)
    cache.append(0, rows, rows)
    path = torch.tensor([[0, 3], [2, -1]], dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="refused"):
        cache.keep(path, torch.tensor([2, 1], dtype=torch.int32, device=dev))
    assert cache.host_lens.tolist() == [42, 41] == cache.seq_lens.tolist()
    assert cache.keep(path[:, :1] * 0, torch.ones(2, dtype=torch.int32, device=dev)).tolist() == [1, 1]
    assert cache.host_lens.tolist() == [41, 41] and int(cache.free_top.item()) == cache.host_free


@pytest.mark.parametrize("counts", [6, np.array([6, 4, 0])])
def test_a_keep_after_a_release(dev, counts) -> None:
    """A released sequence has no newest tokens, whether all had as many or each its own."""
    from saint_kv import Fp4TokenCache

    rng = np.random.default_rng(7)
    cache = Fp4TokenCache(1, 3, 128, 1, 32, block_size=16, device=dev)
    for n in (np.array([20, 30, 16]), counts):
        cache.reserve(n)
        t = int(np.max(n))
        cache.append(0, rows_of(dev, rng, 3, t, 1, 32), rows_of(dev, rng, 3, t, 1, 32))
    cache.release(np.array([True, False, False]))
    third = 0 if isinstance(counts, np.ndarray) else 1
    path = torch.tensor([[-1, -1], [1, 3], [5, -1]], dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="refused"):
        cache.keep(path * 0, torch.tensor([1, 2, third], dtype=torch.int32, device=dev))
    for n_keep in ([0, 2, third], [0, 1, 0]):  # and of those that stayed
        assert cache.keep(path, torch.tensor(n_keep, dtype=torch.int32, device=dev)).tolist() == n_keep
        path = path * 0
    assert cache.host_lens.tolist() == [0, 31, 16] == cache.seq_lens.tolist()
    assert int(cache.free_top.item()) == cache.host_free
