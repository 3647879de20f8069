"""Attention over the 4-bit pages of drafted trees, and of windows whose first tokens stay visible, against the formula in
64 bits on the very bytes of the pages.

Tolerance, per output: a weight is rounded to bf16 for its product with a value (half a step: 2^-8 of each term, so 2^-8 of
A = sum w |v| / (sum w + sink)), the output once (2^-8 of it); scores, sums and exponentials are fp32 and err by less than a
quarter of a bf16 half step for the scores here (|s| < 60): 2^-8 |want| + 1.25 * 2^-8 A.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp4_cache as ora

pytestmark = pytest.mark.gpu


def make(dev, lens, block, heads, dim, seed=0, spare=1):
    """Pages of normally distributed tokens among stale ones (every scale byte NaN's), a shuffled table."""
    from saint_kv import ops

    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, dtype=np.int32)
    pages = -(-lens // block)
    n_pages = int(pages.sum()) + 2
    pool = ops.fp4_pool(n_pages, block, heads, dim, dev)
    pool.fill_(0xFF)
    bt = np.full((len(lens), max(1, int(pages.max(initial=0))) + spare), -1, dtype=np.int32)
    order, at = rng.permutation(n_pages).astype(np.int32), 0
    for b, p in enumerate(pages):
        bt[b, :p] = order[at:at + p]
        at += p
    bt_t, lens_t = torch.as_tensor(bt, device=dev), torch.as_tensor(lens, device=dev)
    t = max(1, int(lens.max(initial=0)))
    g = torch.Generator(device=dev).manual_seed(seed)
    k, v = (torch.randn(len(lens), t, heads, dim, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    ops.fp4_quant_append(pool, bt_t, lens_t, k, v, lens_t)
    return pool, bt_t, lens_t


def masks(batch: int, t: int, n_new, seed: int) -> np.ndarray:
    """bool [B, T, T]: trees with a few roots; in a larger one a node in the middle that sees nothing."""
    rng = np.random.default_rng(seed)
    parents = np.full((batch, t), -1, dtype=np.int32)
    for b in range(batch):
        for i in range(1, t):
            near = rng.integers(max(0, i - 3), i) if rng.random() < 0.7 else rng.integers(0, i)
            parents[b, i] = -1 if rng.random() < 0.06 else near
    seen = ora.tree_masks(parents, np.asarray(n_new))
    if t > 5:
        seen[-1, t // 2] = False
    return seen


def to_words(seen: np.ndarray, dev) -> torch.Tensor:
    """The words of the masks, with bits of later tokens that are not to be read."""
    t = seen.shape[2]
    later = np.arange(t)[None, :] > np.arange(t)[:, None]
    rng = np.random.default_rng(1)
    junk = later & (rng.random((t, t)) < 0.5)
    empty = ~seen.any(-1, keepdims=True)
    return torch.as_tensor(ora.pack_masks(seen | (junk & ~empty)), device=dev)


def check(got, q, pool, bt, lens, **kw):
    """One output, or several of the same call."""
    qn, pn, btn, ln = q.cpu().double().numpy(), pool.cpu().numpy(), bt.cpu().numpy(), lens.cpu().numpy()
    kw = {n: x.cpu().numpy() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    want = ora.view_attention(qn, pn, btn, ln, **kw)
    mag = pn.copy()
    p = ora.Pages(mag)
    half = p.block * p.dim // 2
    p.flat[:, :, half:2 * half] &= 0x77  # |v|: the signs of the values' codes cleared
    a = ora.view_attention(qn, mag, btn, ln, **kw)
    for i, one in enumerate(got if isinstance(got, list) else [got]):
        g = one.detach().cpu().double().numpy().reshape(want.shape)
        assert np.array_equal(np.isnan(g), np.isnan(want))
        off = np.abs(g - want) - (2.0 ** -8 * np.abs(want) + 1.25 * 2.0 ** -8 * a)
        off[np.isnan(want)] = -1
        assert (off <= 0).all(), f"output {i}: worst {off.max()} at {np.unravel_index(off.argmax(), off.shape)}"


TREES = [
    # lens, n_new (None: all), T, H, Hkv, D, block, window, first, sink, softcap
    ([1], None, 1, 1, 1, 32, 16, None, 0, False, None),
    ([333], None, 8, 16, 2, 128, 16, None, 0, False, None),
    ([8, 9, 40, 31, 33], [8, 7, 8, 0, 3], 8, 4, 1, 64, 16, None, 0, True, None),
    ([5, 2, 0, 12], None, 6, 4, 2, 96, 16, None, 0, False, None),  # shorter than their new tokens, or just as long
    ([200, 150, 70], [33, 20, 33], 33, 3, 1, 128, 32, None, 0, False, 20.0),
    ([300, 129, 64], [64, 60, 64], 64, 8, 4, 64, 64, None, 0, True, None),
    ([300, 65, 90], [65, 65, 1], 65, 2, 1, 160, 16, None, 0, False, None),
    ([500, 140], [130, 129], 130, 4, 2, 128, 128, None, 0, False, None),
    ([420, 300], None, 300, 2, 1, 64, 16, None, 0, False, None),
    ([400, 90, 33], [20, 20, 9], 20, 16, 1, 512, 16, None, 0, True, 30.0),
    ([300, 129], [40, 40], 40, 6, 2, 256, 48, None, 0, False, None),
    ([200, 90, 41, 12], [12, 12, 12, 11], 12, 4, 2, 128, 16, 33, 0, False, None),
    ([200, 90, 41, 12], [12, 12, 12, 11], 12, 4, 2, 128, 16, 33, 5, False, None),
    ([200, 99, 64], [60, 60, 60], 60, 2, 1, 64, 16, 3, 2, True, None),  # windows of a part of a path
    ([200, 99, 64], [60, 60, 60], 60, 2, 1, 64, 16, 1, 0, False, None),
    ([200, 99, 64, 70], [60, 60, 60, 66], 66, 2, 1, 64, 16, 2, 7, False, None),  # first tokens that are drafted ones
    ([600, 300], [99, 99], 99, 16, 1, 512, 16, 128, 40, True, 30.0),
    ([1500, 700], [5, 5], 5, 12, 3, 224, 16, 64, 500, False, None),
    ([800, 100], [70, 33], 70, 4, 2, 32, 16, 200, 100, False, None),
]


@pytest.mark.parametrize("lens,n_new,t,heads,kv,dim,block,window,first,sink,softcap", TREES)
def test_trees(dev, lens, n_new, t, heads, kv, dim, block, window, first, sink, softcap) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens_t = make(dev, lens, block, kv, dim, seed=dim + t)
    g = torch.Generator(device=dev).manual_seed(t)
    q = torch.randn(len(lens), t, heads, dim, generator=g, device=dev).to(torch.bfloat16)
    seen = masks(len(lens), t, n_new or [t] * len(lens), seed=t)
    n_new = None if n_new is None else torch.tensor(n_new, dtype=torch.int32, device=dev)
    kw = dict(window=window, softcap=softcap, sink=torch.randn(heads, generator=g, device=dev) if sink else None,
              n_new=n_new, first=first)
    tree = to_words(seen, dev)
    every = [fp4_attention(q, pool, bt, lens_t, splits=splits, tree=tree, **kw) for splits in (0, 1, 3)]
    got = every[-1]
    assert got.dtype == torch.bfloat16 and got.shape == q.shape
    check(every, q, pool, bt, lens_t, seen=seen, **kw)
    if t == 1:
        assert torch.equal(fp4_attention(q[:, 0], pool, bt, lens_t, splits=3, tree=tree, **kw), got[:, 0])


STREAMS = [
    # lens, n_new, T, H, Hkv, D, block, window, first, sink, softcap
    ([1, 5, 0, 700], None, 1, 4, 2, 128, 16, 3, 2, False, None),
    ([333, 90, 33, 34, 35, 36], None, 1, 8, 1, 64, 16, 32, 2, True, None),
    ([500, 129, 128, 64], None, 1, 16, 1, 512, 16, 64, 4, True, 30.0),
    ([900, 300], None, 1, 12, 3, 96, 64, 1, 1, False, None),
    ([900, 300], None, 1, 6, 2, 160, 32, 100, 333, False, None),  # more first tokens than window
    ([700, 150, 3, 40], None, 4, 8, 4, 128, 32, 17, 33, False, 20.0),
    ([600, 150, 40], [33, 20, 0], 33, 16, 2, 64, 64, 40, 31, True, None),
    ([700, 130], None, 130, 8, 2, 128, 128, 50, 32, False, None),
    ([500, 77], None, 70, 2, 2, 512, 16, 5, 64, False, None),
    ([800], None, 65, 17, 1, 32, 16, 90, 65, True, 5.0),
    ([600, 513], None, 40, 8, 2, 192, 64, 128, 1, False, None),
    ([600, 100], None, 200, 2, 1, 256, 16, 150, 90, False, None),  # tokens before the sequence's start
]


@pytest.mark.parametrize("lens,n_new,t,heads,kv,dim,block,window,first,sink,softcap", STREAMS)
def test_first_tokens(dev, lens, n_new, t, heads, kv, dim, block, window, first, sink, softcap) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens_t = make(dev, lens, block, kv, dim, seed=dim + t)
    g = torch.Generator(device=dev).manual_seed(t)
    q = torch.randn(len(lens), t, heads, dim, generator=g, device=dev).to(torch.bfloat16)
    n_new = None if n_new is None else torch.tensor(n_new, dtype=torch.int32, device=dev)
    kw = dict(window=window, softcap=softcap, sink=torch.randn(heads, generator=g, device=dev) if sink else None,
              n_new=n_new, first=first)
    every = [fp4_attention(q, pool, bt, lens_t, splits=splits, **kw) for splits in (0, 1, 3)]
    got = every[-1]
    check(every, q, pool, bt, lens_t, **kw)
    if t == 1:
        assert torch.equal(fp4_attention(q[:, 0], pool, bt, lens_t, splits=3, **kw), got[:, 0])


@pytest.mark.parametrize("t,heads,kv,dim,window,first,max_len", [
    (8, 8, 4, 128, None, 0, 0), (8, 64, 8, 64, None, 0, 5000), (40, 8, 1, 128, None, 0, 100), (3, 16, 1, 512, None, 0, 5000),
    (40, 4, 1, 128, 2000, 40, 5000), (1, 8, 1, 128, 3000, 700, 0)])
def test_long_sequences_over_several_workgroups(dev, t, heads, kv, dim, window, first, max_len) -> None:
    from saint_kv import fp4_attention

    lens = [4800, 100, 0, 2049]
    pool, bt, lens_t = make(dev, lens, 64, kv, dim, seed=5, spare=40)
    q = torch.randn(4, t, heads, dim, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    seen = masks(4, t, [t] * 4, seed=3)
    tree = to_words(seen, dev)
    kw = dict(window=window, first=first)
    got = fp4_attention(q, pool, bt, lens_t, max_len=max_len, tree=tree, **kw)
    check(got, q, pool, bt, lens_t, seen=seen, **kw)
    assert torch.equal(got, fp4_attention(q, pool, bt, lens_t, max_len=max_len, tree=tree, **kw))  # no order that changes
    check(fp4_attention(q, pool, bt, lens_t, max_len=max_len, **kw), q, pool, bt, lens_t, **kw)


@pytest.mark.parametrize("t,heads,dim", [(4, 4, 128), (33, 8, 64), (5, 4, 512)])
def test_a_chain_is_as_no_tree(dev, t, heads, dim) -> None:
    """Masks of every token up to itself: the same positions as without (the bits may differ: rows and tiles are split
    otherwise, so the fp32 sums run in another order and some weights keep more bits)."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [700, 90, t], 16, 2, dim, seed=4)
    q = torch.randn(3, t, heads, dim, device=dev).to(torch.bfloat16)
    tree = torch.as_tensor(ora.pack_masks(np.broadcast_to(np.tri(t, dtype=bool), (3, t, t))), device=dev)
    for kw in ({}, dict(window=50), dict(window=3, softcap=9.0)):
        for splits in (0, 2):
            check(fp4_attention(q, pool, bt, lens, tree=tree, splits=splits, **kw), q, pool, bt, lens, **kw)
    # first tokens without a window are among those seen anyway
    assert torch.equal(fp4_attention(q, pool, bt, lens, first=9, splits=2), fp4_attention(q, pool, bt, lens, splits=2))
    check(fp4_attention(q, pool, bt, lens, first=9), q, pool, bt, lens)


@pytest.mark.parametrize("t,heads,dim", [(6, 4, 128), (40, 8, 64), (5, 4, 512)])
def test_nan_blocks_reach_only_the_tokens_that_see_them(dev, t, heads, dim) -> None:
    """Of a drafted token among its tree's, of a first token, of one between the first and the window."""
    from saint_kv import fp4_attention, ops

    lens = [300, 300, 300]
    pool, bt, lens_t = make(dev, lens, 16, 1, dim, seed=3)
    for b, pos, which in ((0, 300 - t + 2, 0), (1, 3, 1), (2, 100, 1)):
        x = torch.randn(3, 1, 1, dim, device=dev).to(torch.bfloat16)
        y = x.clone()
        (x if which == 0 else y)[b, 0, 0, dim - 1] = float("nan")
        at, n = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
        at[b], n[b] = pos + 1, 1
        ops.fp4_quant_append(pool, bt, at, x, y, n)
    q = torch.randn(3, t, heads, dim, device=dev).to(torch.bfloat16)
    seen = masks(3, t, [t] * 3, seed=8)
    seen[0, 3] = False  # sees none: 0, not NaN
    tree = to_words(seen, dev)
    got = fp4_attention(q, pool, bt, lens_t, tree=tree)
    check(got, q, pool, bt, lens_t, seen=seen)
    got = fp4_attention(q, pool, bt, lens_t, tree=tree, window=60, first=4)
    check(got, q, pool, bt, lens_t, seen=seen, window=60, first=4)
    assert torch.isnan(got[1]).any() and not torch.isnan(got[2]).any()
    got = fp4_attention(q, pool, bt, lens_t, window=60, first=3)
    check(got, q, pool, bt, lens_t, window=60, first=3)
    assert not torch.isnan(got[1:]).any()


def test_unmapped_pages_are_not_seen(dev) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [250, 100, 60], 16, 1, 64, seed=4)
    bt[0, 0], bt[0, 14], bt[0, 15] = -1, pool.shape[0], -1
    bt[1, :] = -7
    q = torch.randn(3, 20, 4, 64, device=dev).to(torch.bfloat16)
    seen = masks(3, 20, [20] * 3, seed=2)
    got = fp4_attention(q, pool, bt, lens, tree=to_words(seen, dev), window=100, first=20)
    check(got, q, pool, bt, lens, seen=seen, window=100, first=20)
    assert (got[1] == 0).all()


def test_nan_queries_of_tokens_that_see_nothing(dev) -> None:
    """A token with an empty mask gives 0, whatever its query holds, and no other token is touched by it."""
    from saint_kv import fp4_attention

    for heads in (4, 16):
        pool, bt, lens = make(dev, [500], 16, 2, 128, seed=4)
        q = torch.randn(1, 30, heads, 128, device=dev).to(torch.bfloat16)
        seen = masks(1, 30, [30], seed=2)
        seen[0, 7] = False
        clean = fp4_attention(q, pool, bt, lens, tree=to_words(seen, dev))
        q[0, 7] = float("nan")
        got = fp4_attention(q, pool, bt, lens, tree=to_words(seen, dev))
        assert (got[0, 7] == 0).all() and torch.equal(got, clean)


def test_strided_queries_and_given_buffers(dev) -> None:
    from saint_kv import fp4_attention
    from saint_kv.fp4 import fp4_attention_workspace

    pool, bt, lens = make(dev, [900, 450], 64, 2, 128, seed=6)
    q = torch.randn(2, 8, 3, 128, device=dev).to(torch.bfloat16).transpose(1, 2)  # held as [B, H, T, D]
    tree = to_words(masks(2, 3, [3, 3], seed=1), dev)
    for kw in (dict(tree=tree), dict(window=500, first=9)):
        got = fp4_attention(q, pool, bt, lens, splits=4, **kw)
        assert torch.equal(got, fp4_attention(q.contiguous(), pool, bt, lens, splits=4, **kw))
        need = fp4_attention_workspace(q, pool, bt, splits=4, **kw)
        assert need > 16
        out = torch.full_like(got, 3.0)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        assert fp4_attention(q, pool, bt, lens, splits=4, out=out, workspace=ws, **kw) is out
        assert torch.equal(out, got)
        with pytest.raises(ValueError, match="workspace"):
            fp4_attention(q, pool, bt, lens, splits=4, workspace=ws[:need - 16], **kw)


def test_refusals(dev) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [40, 40], 16, 2, 64)
    q = torch.zeros(2, 70, 4, 64, dtype=torch.bfloat16, device=dev)
    tree = torch.zeros(2, 70, 2, dtype=torch.int64, device=dev)
    fp4_attention(q, pool, bt, lens, tree=tree, first=3)
    for bad in (dict(tree=tree.int()), dict(tree=tree[:, :, :1]), dict(tree=tree[:1]), dict(tree=tree[:, :69]),
                dict(tree=torch.zeros(2, 70, 4, dtype=torch.int64, device=dev)[..., ::2]), dict(first=-1),
                dict(first=(1 << 24) + 1), dict(tree=tree[0])):
        with pytest.raises(ValueError):
            fp4_attention(q, pool, bt, lens, **bad)
    with pytest.raises(ValueError, match="tree"):
        fp4_attention(torch.zeros(1, 1025, 2, 64, dtype=torch.bfloat16, device=dev), pool, bt[:1], lens[:1],
                      tree=torch.zeros(1, 1025, 17, dtype=torch.int64, device=dev))
    with pytest.raises(RuntimeError, match="CPU"):
        fp4_attention(q, pool, bt, lens, tree=tree.cpu())


def test_captured_attention_replays(dev) -> None:
    """A tree's and a window's graph, replayed in turn over lengths and masks that eager work changes."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [2000, 700], 64, 1, 128, seed=8)
    q = torch.zeros(2, 9, 8, 128, dtype=torch.bfloat16, device=dev)
    q1 = torch.zeros(2, 1, 8, 128, dtype=torch.bfloat16, device=dev)
    tree = to_words(masks(2, 9, [9, 9], seed=1), dev)
    calls = [(q, dict(tree=tree)), (q1, dict(window=900, first=70))]
    for x, kw in calls:
        fp4_attention(x, pool, bt, lens, **kw)
    torch.cuda.synchronize()
    graphs = []
    for x, kw in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp4_attention(x, pool, bt, lens, **kw)
        graphs.append((graph, x, kw, y))
    for n in range(4):
        lens.copy_(torch.tensor([2000 - 700 * (n % 2), 700 - 90 * n], dtype=torch.int32))
        tree.copy_(to_words(masks(2, 9, [9, 9], seed=n), dev))
        for graph, x, _, _ in graphs:
            x.copy_(torch.randn(x.shape, device=dev))
            graph.replay()
        torch.cuda.synchronize()
        for _, x, kw, y in graphs:
            assert torch.equal(y, fp4_attention(x, pool, bt, lens, **kw))


def test_far_pages(dev) -> None:
    """Pages past 4 GiB of the pool."""
    from saint_kv import fp4_attention, ops

    heads, dim, block = 8, 512, 128
    n_pages = (5 << 30) // (block * heads * dim * 17 // 16)
    pool = torch.empty(n_pages, block, heads, 17 * dim // 16, dtype=torch.uint8, device=dev)
    bt = torch.tensor([[n_pages - 1, 0], [n_pages - 2, n_pages - 3]], dtype=torch.int32, device=dev)
    lens = torch.tensor([200, 131], dtype=torch.int32, device=dev)
    k, v = (torch.randn(2, 200, heads, dim, device=dev).to(torch.bfloat16) for _ in range(2))
    ops.fp4_quant_append(pool, bt, lens, k, v, lens)
    q = torch.randn(2, 4, heads, dim, device=dev).to(torch.bfloat16)
    seen = masks(2, 4, [4, 4], seed=1)
    got = fp4_attention(q, pool, bt, lens, tree=to_words(seen, dev), window=90, first=3)
    ids = torch.unique(bt).long()
    small = torch.searchsorted(ids, bt.long()).to(torch.int32)
    check(got, q, pool[ids], small, lens, seen=seen, window=90, first=3)


@pytest.mark.parametrize("t,heads,kv,dim,sink", [(70, 16, 2, 96, True), (70, 16, 2, 128, False), (40, 16, 2, 256, True), (90, 16, 2, 64, False)])
def test_many_rows_in_parts(dev, t, heads, kv, dim, sink) -> None:
    """Cut items of shared tiles with so many rows that a workgroup joins an item's blocks; a NaN block among the old tokens."""
    from saint_kv import fp4_attention, ops

    lens = [1400, 300, 5, 700]
    pool, bt, lens_t = make(dev, lens, 16, kv, dim, seed=dim, spare=60)
    x = torch.randn(4, 1, kv, dim, device=dev).to(torch.bfloat16)
    y = x.clone()
    y[1, 0, 1, 3] = float("inf")
    at, one = torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    at[1], one[1] = 40, 1
    ops.fp4_quant_append(pool, bt, at, x, y, one)
    q = torch.randn(4, t, heads, dim, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    kw = dict(sink=torch.linspace(-3, 3, heads, device=dev) if sink else None)
    seen = masks(4, t, [t] * 4, seed=3)
    got = fp4_attention(q, pool, bt, lens_t, tree=to_words(seen, dev), **kw)
    check(got, q, pool, bt, lens_t, seen=seen, **kw)
    assert torch.isnan(got[1]).any() and not torch.isnan(got[0]).any() and (got[2] == 0).all()
    check(fp4_attention(q, pool, bt, lens_t, window=600, first=20, **kw), q, pool, bt, lens_t, window=600, first=20, **kw)


def test_calls_on_two_streams_at_once(dev) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [3000, 900], 64, 2, 128, seed=6, spare=20)
    tree = to_words(masks(2, 6, [6, 6], seed=1), dev)
    calls = [(torch.randn(2, 6, 8, 128, device=dev).to(torch.bfloat16), dict(tree=tree)),
             (torch.randn(2, 1, 8, 128, device=dev).to(torch.bfloat16), dict(window=2000, first=100)),
             (torch.randn(2, 6, 64, 128, device=dev).to(torch.bfloat16), dict(tree=tree, window=900, first=5))]
    want = [fp4_attention(q, pool, bt, lens, **kw) for q, kw in calls]
    streams = [torch.cuda.Stream(device=dev) for _ in calls]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream, (q, kw) in zip(streams, calls):
            with torch.cuda.stream(stream):
                got.append(fp4_attention(q, pool, bt, lens, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 3]) for i, g in enumerate(got))


@pytest.mark.parametrize("seed", range(12))
def test_random_views(dev, seed) -> None:
    """Shapes, windows, trees and lengths at random, small enough for the oracle."""
    from saint_kv import fp4_attention

    rng = np.random.default_rng(100 + seed)
    batch, kv, g = int(rng.integers(1, 5)), int(rng.integers(1, 4)), int(rng.integers(1, 9))
    dim, block = int(rng.choice([32, 64, 96, 128, 192, 256, 384, 512])), int(rng.choice([16, 48, 64]))
    t = int(rng.choice([1, 3, 17, 40, 66]))
    lens = rng.integers(0, 400, batch)
    n_new = rng.integers(0, t + 1, batch).astype(np.int32)
    pool, bt, lens_t = make(dev, lens, block, kv, dim, seed=seed)
    q = torch.randn(batch, t, kv * g, dim, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(torch.bfloat16)
    kw = dict(window=int(rng.integers(1, 200)) if rng.random() < 0.7 else None, first=int(rng.integers(0, 80)),
              n_new=torch.as_tensor(n_new, device=dev) if rng.random() < 0.6 else None, softcap=20.0 if rng.random() < 0.3 else None,
              sink=torch.randn(kv * g, device=dev) if rng.random() < 0.5 else None)
    seen = masks(batch, t, n_new if kw["n_new"] is not None else [t] * batch, seed)
    more = dict(max_len=int(rng.choice([0, 50, 400])), splits=int(rng.choice([0, 0, 2])))
    check(fp4_attention(q, pool, bt, lens_t, tree=to_words(seen, dev), **kw, **more), q, pool, bt, lens_t, seen=seen, **kw)
    check(fp4_attention(q, pool, bt, lens_t, **kw, **more), q, pool, bt, lens_t, **kw)


@pytest.mark.parametrize("lens,n_new,t,heads,kv,block,window,first,sink,softcap", [
    ([1500, 700, 33, 0, 40], [40, 33, 33, 0, 1], 40, 16, 1, 16, None, 0, False, None),
    ([1500, 700, 45, 0, 39], None, 40, 16, 1, 64, 200, 70, True, 30.0),
    ([130, 64, 65, 31, 32, 1, 100, 99], None, 1, 80, 2, 16, None, 0, True, None),  # 40 rows a head
    ([300] * 17, None, 3, 11, 1, 16, 100, 4, False, None),  # 33 rows
    ([1900, 1300], None, 66, 16, 2, 64, None, 0, False, 5.0)])
def test_wide_heads_whose_waves_share_tiles(dev, lens, n_new, t, heads, kv, block, window, first, sink, softcap) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens_t = make(dev, lens, block, kv, 512, seed=t)
    g = torch.Generator(device=dev).manual_seed(t)
    q = torch.randn(len(lens), t, heads, 512, generator=g, device=dev).to(torch.bfloat16)
    seen = masks(len(lens), t, n_new or [t] * len(lens), seed=t)
    counts = None if n_new is None else torch.tensor(n_new, dtype=torch.int32, device=dev)
    kw = dict(window=window, softcap=softcap, sink=torch.randn(heads, generator=g, device=dev) if sink else None,
              n_new=counts, first=first)
    for tree, of in ((to_words(seen, dev), seen), (None, None)):
        if tree is None and not first:
            continue
        extra = {} if of is None else {"seen": of}
        every = [fp4_attention(q, pool, bt, lens_t, splits=splits, tree=tree, **kw) for splits in (0, 1, 3)]
        check(every, q, pool, bt, lens_t, **extra, **kw)
        for splits, got in zip((0, 1, 3), every):
            assert torch.equal(got, fp4_attention(q, pool, bt, lens_t, splits=splits, tree=tree, **kw))


@pytest.mark.parametrize("lens,t,heads,kv,dim", [([333], 8, 16, 2, 128), ([300] * 17, 3, 11, 1, 512), ([1500, 700], 40, 16, 1, 512),
                                                 ([200, 90, 41, 12], 5, 12, 3, 224), ([900, 0, 5], 1, 8, 1, 64)])
def test_first_tokens_without_a_window_are_no_view(dev, lens, t, heads, kv, dim) -> None:
    """Every position is seen with them and without: the plain call, to the bit, and its workspace."""
    from saint_kv import fp4_attention
    from saint_kv.fp4 import fp4_attention_workspace

    pool, bt, lens_t = make(dev, lens, 16, kv, dim, seed=2)
    q = torch.randn(len(lens), t, heads, dim, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    for splits in (0, 3):
        got = fp4_attention(q, pool, bt, lens_t, first=4, splits=splits)
        assert torch.equal(got, fp4_attention(q, pool, bt, lens_t, splits=splits))
        need = [fp4_attention_workspace(q, pool, bt, first=first, splits=splits) for first in (0, 4)]
        assert need[0] == need[1]


def some(keep, q, pool, bt, lens, seen):
    """Of a large batch the sequences of a sample: what check takes of them, their pages alone."""
    ids, small = torch.unique(bt[keep].clamp_min(0).long(), return_inverse=True)
    table = torch.where(bt[keep] < 0, -1, small.to(torch.int32))
    return q[keep], pool[ids], table, lens[keep], seen[keep.cpu().numpy()]


@pytest.mark.parametrize("batch", [100, 300])
def test_pieces_of_many_sequences(dev, batch) -> None:
    """More items than a workgroup counts in one turn, or than a wave looks through at once, each in pieces of its own."""
    from saint_kv import fp4_attention

    rng = np.random.default_rng(batch)
    lens = rng.integers(600, 1500, batch)
    lens[[0, 7, batch // 2, batch - 1]] = [0, 2, 33, 0]
    pool, bt, lens_t = make(dev, lens, 64, 1, 64, seed=1)
    q = torch.randn(batch, 2, 2, 64, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    seen = masks(batch, 2, [2] * batch, seed=4)
    got = fp4_attention(q, pool, bt, lens_t, tree=to_words(seen, dev))
    assert torch.equal(got, fp4_attention(q, pool, bt, lens_t, tree=to_words(seen, dev)))
    keep = torch.unique(torch.cat((torch.tensor([0, 1, 7, 63, 64, batch // 2, batch - 2, batch - 1]),
                                   torch.as_tensor(rng.integers(0, batch, 24))))).to(dev)
    q, pool, bt, lens_t, seen = some(keep, q, pool, bt, lens_t, seen)
    check(got[keep], q, pool, bt, lens_t, seen=seen)


@pytest.mark.parametrize("lens,t,heads,kv,dim,window,first", [
    ([2600, 1800, 1700, 1000, 33, 0] + [2500] * 58, 1, 8, 8, 128, 1600, 4),  # 51 tiles
    ([5200, 4900, 4700, 3000] + [5000] * 92, 1, 8, 8, 64, 4700, 70),  # 152
    ([2400, 2300, 900], 512, 32, 32, 128, 1700, 40), ([3500, 3000, 1000] + [2900] * 21, 64, 16, 8, 256, 2700, 1)])
def test_windows_left_whole(dev, lens, t, heads, kv, dim, window, first) -> None:
    """Windows of 49 to 160 tiles that are not cut: no workspace, one launch."""
    from saint_kv import fp4_attention
    from saint_kv.fp4 import fp4_attention_workspace

    batch = len(lens)
    pool, bt, lens_t = make(dev, lens, 64, kv, dim, seed=t)
    q = torch.randn(batch, t, heads, dim, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    assert fp4_attention_workspace(q, pool, bt, window=window, first=first) == 0
    got = fp4_attention(q, pool, bt, lens_t, window=window, first=first)
    keep = torch.arange(min(batch, 4 if t == 1 else 3), device=dev)
    step = max(1, t // 3)  # rows of a chunk: its newest, and others down to its oldest
    rows = torch.arange(t - 1, -1, -step).flip(0)
    q, pool, bt, lens_t, _ = some(keep, q, pool, bt, lens_t, np.zeros((batch, 1, 1)))
    for r in rows.tolist():  # as the newest of a sequence that ends with it
        check(got[keep, r:r + 1], q[:, r:r + 1], pool, bt, lens_t - (t - 1 - r), window=window, first=first)
