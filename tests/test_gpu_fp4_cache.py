"""The 4-bit cache's operators run together, as a model's layers do, and the forms
of its attention that the lengths, rows and splits choose between, against the
plain 64-bit attention over the same bytes.

Bounds are those of test_gpu_fp4_attention.py: weights and output rounded to bf16
once each (2^-8 of the weighted |v| sum and of the output), with a quarter more of
the first for the two's crossing and the fp32 sums.  What two runs of the same
kernels on the same bytes give is equal to the bit.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_fp4_attention import check, make

from oracle import fp4_cache as ora

pytestmark = pytest.mark.gpu


def queries(dev, *shape, seed=0) -> torch.Tensor:
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=dev).to(torch.bfloat16)


# rows of a K/V head: a token's own (1), a few waves' (17..64), shared tiles (65 on)
@pytest.mark.parametrize("t,heads,kv,dim,sink,window", [
    (3, 4, 2, 64, False, None), (9, 6, 2, 96, True, None), (40, 16, 4, 128, True, None), (70, 4, 2, 64, True, 20),
    (70, 2, 1, 256, False, None), (33, 4, 2, 512, True, None), (65, 8, 2, 128, False, 48)])
def test_padded_batch(dev, t, heads, kv, dim, sink, window) -> None:
    """Each sequence's first n_new tokens are its own, none of some; the others' outputs are zeros."""
    from saint_kv import fp4_attention

    lens = [200, 1, 33, 64, 90]
    n_new = np.minimum([t, 1, 0, t - 1, 2], lens).astype(np.int32)
    pool, bt, lens_t = make(dev, lens, 16, kv, dim, seed=t)
    q = queries(dev, len(lens), t, heads, dim, seed=dim)
    s = torch.linspace(-2, 2, heads, device=dev) if sink else None
    got = fp4_attention(q, pool, bt, lens_t, n_new=torch.as_tensor(n_new, device=dev), sink=s, window=window)
    check(got, q, pool, bt, lens_t, n_new=n_new, sink=s, window=window)
    for b, n in enumerate(n_new):
        assert not got[b, n:].any()


def test_counts_outside_the_queries(dev) -> None:
    """A count below zero is none, one past q's tokens all of them."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [50, 60], 16, 1, 64)
    q = queries(dev, 2, 4, 2, 64)
    i32 = dict(dtype=torch.int32, device=dev)
    got = fp4_attention(q, pool, bt, lens, n_new=torch.tensor([-3, 9], **i32))
    want = fp4_attention(q, pool, bt, lens, n_new=torch.tensor([0, 4], **i32))
    assert torch.equal(got, want) and torch.equal(want[1], fp4_attention(q, pool, bt, lens)[1])
    for bad in (torch.tensor([1, 2], device=dev), torch.tensor([1], **i32)):
        with pytest.raises(ValueError):
            fp4_attention(q, pool, bt, lens, n_new=bad)
    with pytest.raises(RuntimeError):
        fp4_attention(q, pool, bt, lens, n_new=torch.tensor([1, 2], dtype=torch.int32))


@pytest.mark.parametrize("splits", [1, 2, 5, 40])
@pytest.mark.parametrize("t,heads,kv,dim", [(1, 4, 2, 128), (3, 12, 1, 96), (1, 3, 1, 512), (40, 4, 2, 64), (70, 1, 1, 256)])
def test_splits(dev, t, heads, kv, dim, splits) -> None:
    """Any cut of the sequences, also into more parts than they have tiles."""
    from saint_kv import fp4_attention

    lens = [700, 0, 31, 400]
    pool, bt, lens_t = make(dev, lens, 16, kv, dim, seed=splits)
    q = queries(dev, len(lens), t, heads, dim, seed=t)
    check(fp4_attention(q, pool, bt, lens_t, splits=splits), q, pool, bt, lens_t)


@pytest.mark.parametrize("batch,kv,lens", [(2100, 1, (0, 40)), (112, 8, (600, 610)), (100, 8, (0, 900))])
def test_many_sequences(dev, batch, kv, lens) -> None:
    """More sequences than are dealt out in runs, as many of one length as there are
    workgroups, and ragged ones."""
    from saint_kv import fp4_attention

    n = np.random.default_rng(batch).integers(*lens, size=batch)
    pool, bt, lens_t = make(dev, n, 16, kv, 32, seed=batch, spare=40)
    q = queries(dev, batch, 1, kv, 32)
    check(fp4_attention(q, pool, bt, lens_t), q, pool, bt, lens_t)


def test_many_row_blocks(dev) -> None:
    """Whole prompts: more row blocks than are dealt out in runs, against the rows read back."""
    from saint_kv import fp4_attention, ops

    batch, t, heads, dim = 9, 2048, 16, 32
    lens = [2048 + 7 * b for b in range(batch)]
    pool, bt, lens_t = make(dev, lens, 64, 1, dim)
    q = queries(dev, batch, t, heads, dim)
    got = fp4_attention(q, pool, bt, lens_t)
    k, v = (torch.zeros(batch, lens[-1], 1, dim, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ops.fp4_gather(pool, bt, lens_t, k, v, lens_t)
    for b, h in ((0, 0), (0, 15), (5, 7), (8, 3)):
        n = lens[b]
        s = (q[b, :, h].double() @ k[b, :n, 0].double().T.contiguous()) * dim ** -0.5
        seen = torch.arange(n, device=dev)[None, :] <= torch.arange(n - t, n, device=dev)[:, None]
        p = torch.softmax(s.masked_fill(~seen, float("-inf")), 1)
        want, a = p @ v[b, :n, 0].double(), p @ v[b, :n, 0].double().abs()
        assert ((got[b, :, h].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.25 * 2.0 ** -8 * a).all()


def test_two_streams_at_once(dev) -> None:
    """Calls in flight together, each with a workspace of its own."""
    from saint_kv import fp4_attention

    work = []
    for n, (t, heads, dim) in enumerate(((1, 8, 128), (80, 4, 64))):
        pool, bt, lens = make(dev, [9000, 3000, 50], 64, 2, dim, seed=n)
        q = queries(dev, 3, t, heads, dim, seed=n)
        work.append((q, pool, bt, lens, fp4_attention(q, pool, bt, lens), torch.cuda.Stream(dev)))
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for q, pool, bt, lens, _, stream in work:
            with torch.cuda.stream(stream):
                got.append(fp4_attention(q, pool, bt, lens))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, work[i % 2][4])


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("t,heads", [(1, 3), (1, 40), (70, 2)])
def test_a_query_that_is_not_finite(dev, t, heads, bad) -> None:
    """Its own outputs are NaN, and no others."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [100, 90], 16, 1, 128)
    q = queries(dev, 2, t, heads, 128)
    want = fp4_attention(q, pool, bt, lens)
    q[1, t - 1, heads - 1, 77] = bad
    got = fp4_attention(q, pool, bt, lens)
    assert torch.isnan(got[1, t - 1, heads - 1]).all()
    got[1, t - 1, heads - 1] = want[1, t - 1, heads - 1]
    assert torch.equal(got, want)


def test_scores_at_the_ends_of_fp32(dev) -> None:
    """Scales that fp32 cannot carry are refused; the largest that it can are right."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [40], 16, 1, 64)
    q = queries(dev, 1, 1, 2, 64)
    for kw in (dict(scale=3e38), dict(softcap=3e38), dict(softcap=1e-38, scale=10.0)):
        with pytest.raises(ValueError):
            fp4_attention(q, pool, bt, lens, **kw)
    check(fp4_attention(q, pool, bt, lens, softcap=1e-30), q, pool, bt, lens, softcap=1e-30)
    check(fp4_attention(q, pool, bt, lens, scale=1e-30), q, pool, bt, lens, scale=1e-30)


# -- a model's layers over Fp4TokenCache ---------------------------------------
LAYERS, HEADS, KV, DIM, BLOCK = 3, 6, 2, 64, 16


class Model:
    """What a stack of layers sends through the cache, from a seed: the same tokens
    of a sequence whatever else the batch does."""

    def __init__(self, dev, cache) -> None:
        self.dev, self.cache, self.tokens = dev, cache, [[] for _ in range(cache.batch)]

    def rows(self, what: int, i: int, t: int) -> torch.Tensor:
        """[B, t, heads, dim] for the tokens reserved last."""
        heads = HEADS if what == 0 else KV
        out = torch.zeros(self.cache.batch, t, heads, DIM)
        for b, (first, n) in enumerate(self.last):
            for j in range(n):
                g = torch.Generator().manual_seed(((self.seed[b] * 1000 + first + j) * LAYERS + i) * 3 + what)
                out[b, j] = torch.randn(heads, DIM, generator=g)
        return out.to(self.dev, torch.bfloat16)

    seed = list(range(64))

    def step(self, counts) -> list[torch.Tensor]:
        n = np.broadcast_to(np.asarray(counts), (self.cache.batch,))
        self.last = [(int(self.cache.host_lens[b]), int(n[b])) for b in range(self.cache.batch)]
        self.cache.reserve(counts)
        t, outs = int(n.max()), []
        for i in range(LAYERS):
            self.cache.append(i, self.rows(1, i, t), self.rows(2, i, t))
            self.q = self.rows(0, i, t)
            outs.append(self.cache.attention(i, self.q))
            check(outs[-1], self.q, self.cache.pool[i], self.cache.block_table, self.cache.seq_lens,
                  n_new=n.astype(np.int32))
        self.cache.check_status()
        return outs


def new_cache(dev, batch=5, pages=None, max_len=160):
    from saint_kv import Fp4TokenCache

    return Fp4TokenCache(LAYERS, batch, max_len, KV, DIM, block_size=BLOCK, n_pages=pages, device=dev)


def test_layers_fork_release_compact(dev) -> None:
    cache = new_cache(dev)
    m = Model(dev, cache)
    m.step([37, 64, 0, 0, 5])
    m.step(np.array([1, 1, 0, 0, 1]))
    used = cache.n_pages - int(cache.free_top)
    cache.fork([0, 1], [2, 3])
    # 38 tokens: two whole pages shared, one begun page copied; 65: four and one
    assert cache.n_pages - int(cache.free_top) == used + 2
    assert cache.host_lens.tolist() == [38, 65, 38, 65, 6]
    m.seed = [0, 1, 0, 1, 4]
    outs = m.step(1)  # the forks get their sources' tokens: their outputs are the same
    for x in outs:
        assert torch.equal(x[0], x[2]) and torch.equal(x[1], x[3])
    m.seed = [0, 1, 7, 9, 4]
    outs = m.step(np.array([3, 1, 2, 20, 1]))  # and go their own ways
    assert not torch.equal(outs[0][0, :2], outs[0][2, :2])
    before = [cache.attention(i, torch.ones(5, 1, HEADS, DIM, dtype=torch.bfloat16, device=dev)) for i in range(LAYERS)]
    cache.release(np.array([True, False, False, False, True]))
    live, moved = cache.compact()
    assert live == cache.n_pages - int(cache.free_top) and moved > 0
    held = cache.block_table[cache.block_table >= 0].unique()
    assert held.numel() == live and int(held.max()) == live - 1  # defragmented
    after = [cache.attention(i, torch.ones(5, 1, HEADS, DIM, dtype=torch.bfloat16, device=dev)) for i in range(LAYERS)]
    for x, y in zip(before, after):
        assert torch.equal(x[1:4], y[1:4])
        assert not y[0].any() and not y[4].any()
    m.step(np.array([18, 1, 1, 1, 0]))  # a new sequence in the slot that is free again
    cache.release(np.array([True, True, True, True, False]))
    assert int(cache.free_top) == cache.n_pages and not cache.refs.any()
    assert sorted(cache.free_stack.tolist()) == list(range(cache.n_pages))


def test_too_few_pages(dev) -> None:
    """What does not fit raises and changes nothing, and the rest goes on."""
    cache = new_cache(dev, pages=4)
    m = Model(dev, cache)
    m.step([20, 20, 0, 0, 0])
    for what in (lambda: cache.reserve([40, 0, 0, 0, 0]), lambda: cache.fork([0], [2])):
        with pytest.raises(RuntimeError, match="out of pages"):
            what()
        assert cache.host_lens.tolist() == cache.seq_lens.tolist() == [20, 20, 0, 0, 0]
    m.step([1, 12, 0, 0, 0])
    cache.release(np.array([1, 0, 0, 0, 0]))
    assert cache.host_free == int(cache.free_top) == 2
    cache.fork([1, 1], [0, 2])  # 32 tokens: whole pages, no copies
    assert cache.host_free == int(cache.free_top) == 2
    m.seed = [1, 1, 1, 3, 4]
    x = m.step([1, 0, 1, 0, 0])[0]
    assert torch.equal(x[0], x[2]) and cache.host_free == int(cache.free_top) == 0
    with pytest.raises(RuntimeError, match="overflow"):
        cache.reserve(160)
    with pytest.raises(RuntimeError, match="empty"):
        cache.fork([0], [1])
    with pytest.raises(RuntimeError, match="double free"):
        cache.release(np.array([0, 0, 0, 1, 0]))
    for bad in (lambda: cache.fork([0], [5]), lambda: cache.fork([0, 1], [3, 3]), lambda: cache.reserve(-1),
                lambda: cache.release(np.array([1, 0]))):
        with pytest.raises(ValueError):
            bad()
    cache.release(np.array([1, 1, 1, 0, 0]))
    assert cache.host_free == cache.n_pages and not cache.refs.any()


def test_on_another_stream(dev) -> None:
    """All of it on a stream that is not the default one, beside other work there."""
    want_cache, cache = new_cache(dev), new_cache(dev)
    a, b = Model(dev, want_cache), Model(dev, cache)
    want = [a.step([30, 2, 17, 0, 64]), a.step(1)]
    busy = torch.randn(2048, 2048, device=dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        got = []
        for counts in ([30, 2, 17, 0, 64], 1):
            busy @ busy  # noqa: B018  (work in front of the step)
            got.append(b.step(counts))
    torch.cuda.current_stream(dev).wait_stream(stream)
    for x, y in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(x, y))


def test_captured_steps(dev) -> None:
    """A step of reservation, write and attention as a graph: replays continue the
    sequences as eager steps of a second cache do, in pages popped on the device."""
    from saint_kv import fp4_attention, ops

    caches = [new_cache(dev), new_cache(dev)]
    for c in caches:
        Model(dev, c).step([15, 16, 1, 40, 0])
    g = torch.Generator(device=dev).manual_seed(3)
    k, v, q = (torch.empty(5, 1, h, DIM, dtype=torch.bfloat16, device=dev) for h in (KV, KV, HEADS))

    def step(c):
        ops.reserve(c.free_stack, c.free_top, c.block_table, c.seq_lens, 1, BLOCK, c.status)
        ops.fp4_quant_append(c.pool[0], c.block_table, c.seq_lens, k, v, 1)
        return fp4_attention(q, c.pool[0], c.block_table, c.seq_lens)

    for x in (k, v, q):
        x.normal_(generator=g)
    for c in caches:  # both caches take the warm-up step
        step(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for _ in range(20):  # past a page's end in every sequence
        for x in (k, v, q):
            x.normal_(generator=g)
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    for x, y in zip((caches[0].seq_lens, caches[0].block_table), (caches[1].seq_lens, caches[1].block_table)):
        assert torch.equal(x, y)
    assert int(caches[0].status) == 0


def test_expanded_rows(dev) -> None:
    """Rows that are one expanded token are written for every position; none can be read into such."""
    from saint_kv import ops

    lens = torch.tensor([20, 33], dtype=torch.int32, device=dev)
    pool, bt, _ = make(dev, [20, 33], 16, 2, 64)
    k, v = (queries(dev, 1, 1, 2, 64, seed=s).expand(2, 33, 2, 64) for s in (1, 2))
    ops.fp4_quant_append(pool, bt, lens, k, v, lens)
    out = [torch.zeros(2, 33, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    ops.fp4_gather(pool, bt, lens, *out, lens)
    for x, y in zip(out, (k, v)):
        codes, scales = ora.quantize(y[0, 0].double().cpu().numpy())
        want = torch.as_tensor(ora.dequantize(codes, scales))
        assert all(torch.equal(x[b, i].double().cpu(), want) for b, n in ((0, 20), (1, 33)) for i in range(n))
        assert not x[0, 20:].any()
    with pytest.raises(ValueError, match="expanded"):
        ops.fp4_gather(pool, bt, lens, k, v, lens)


def test_what_is_read_back_is_what_attention_sees(dev) -> None:
    """fp4_gather's rows, attended over in 64 bits, give fp4_attention's outputs."""
    from saint_kv import fp4_attention, ops

    lens = [77, 130]
    pool, bt, lens_t = make(dev, lens, 32, 2, 96)
    k, v = (torch.zeros(2, 130, 2, 96, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ops.fp4_gather(pool, bt, lens_t, k, v, lens_t)
    q = queries(dev, 2, 1, 4, 96)
    got = fp4_attention(q, pool, bt, lens_t).double().cpu()
    for b, n in enumerate(lens):
        for h in range(4):
            kk, vv = k[b, :n, h // 2].double().cpu(), v[b, :n, h // 2].double().cpu()
            p = torch.softmax(kk @ q[b, 0, h].double().cpu() * 96 ** -0.5, 0)
            want = p @ vv
            assert ((got[b, 0, h] - want).abs() <= 2.0 ** -8 * want.abs() + 1.25 * 2.0 ** -8 * (p @ vv.abs())).all()
    pages = ora.rows(pool.cpu().numpy(), bt.cpu().numpy(), 0, range(77))
    assert np.array_equal(pages[0], k[0, :77].double().cpu().numpy())
