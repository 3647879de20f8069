"""Forked sequences: tables, counts, free stack and pages bit for bit against the oracle over
random histories; refusals that change nothing; the decode cache's forks."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import reference_cpu as ref
from oracle import shared_pages as ora

pytestmark = pytest.mark.gpu


class Both:
    """A page group with pools on the GPU and as the oracle holds it."""

    def __init__(self, dev, batch, width, n_pages, block, rows=(16, 48), seed=0):
        from saint_kv import ops

        self.ops, self.block, self.dev = ops, block, dev
        order = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
        self.stack, self.top = ref.free_stack_init(n_pages, order)
        self.refs, self.lens = np.zeros(n_pages, np.int32), np.zeros(batch, np.int32)
        self.bt = np.full((batch, width), -1, np.int32)
        g = torch.Generator().manual_seed(seed)
        self.pools = [torch.randint(0, 255, (n_pages, block, r), generator=g, dtype=torch.uint8) for r in rows]
        i32 = dict(dtype=torch.int32, device=dev)
        self.d = dict(stack=torch.empty(n_pages, **i32), top=torch.empty(1, **i32), refs=torch.zeros(n_pages, **i32),
                      bt=torch.full((batch, width), -1, **i32), lens=torch.zeros(batch, **i32),
                      status=torch.zeros(1, **i32), ws=torch.zeros(3 * n_pages, **i32), info=torch.zeros(2, **i32))
        ops.free_stack_init(self.d["stack"], self.d["top"], torch.as_tensor(order, device=dev))
        self.dpools = [p.to(dev) for p in self.pools]

    def reserve(self, n):
        d = self.d
        n = np.asarray(n, dtype=np.int32)
        st, self.top = ref.reserve(self.stack, self.top, self.bt, self.lens, n, self.block)
        self.ops.reserve(d["stack"], d["top"], d["bt"], d["lens"], torch.as_tensor(n, device=self.dev), self.block,
                         d["status"])
        assert int(d["status"]) == st

    def fork(self, src, dst, status=0):
        d = self.d
        if not status:
            self.top = ora.fork(self.stack, self.top, self.refs, self.bt, self.lens, src, dst, self.block, self.pools)
        s, t = (torch.as_tensor(np.asarray(x, dtype=np.int32), device=self.dev) for x in (src, dst))
        self.ops.fork(d["stack"], d["top"], d["refs"], d["bt"], d["lens"], s, t, self.block, self.dpools, d["status"])
        assert int(d["status"]) == status

    def release(self, mask, status=0):
        d = self.d
        mask = np.asarray(mask, dtype=np.uint8)
        if not status:
            self.top = ora.release(self.stack, self.top, self.refs, self.bt, self.lens, mask, self.block)
        self.ops.release(d["stack"], d["top"], d["bt"], d["lens"], torch.as_tensor(mask, device=self.dev), self.block,
                         d["status"], refs=d["refs"])
        assert int(d["status"]) == status

    def compact(self):
        d = self.d
        self.stack, self.top, moved = ora.compact(self.pools, self.refs, self.bt, self.lens, self.block)
        self.ops.compact(self.dpools, d["bt"], d["lens"], self.block, d["stack"], d["top"], d["ws"], d["info"],
                         refs=d["refs"])
        assert d["info"].tolist() == [self.refs.shape[0] - self.top, moved]
        assert not d["ws"][:self.refs.shape[0]].any()

    def check(self):
        d = self.d
        assert int(d["top"]) == self.top
        assert np.array_equal(d["stack"].cpu().numpy()[:self.top], self.stack[:self.top])
        for name in ("refs", "bt", "lens"):
            assert np.array_equal(d[name].cpu().numpy(), getattr(self, name)), name
        for a, b in zip(self.dpools, self.pools):
            assert torch.equal(a.cpu(), b)
        ora.check(self.refs, self.stack, self.top, self.bt, self.lens, self.block)


@pytest.mark.parametrize("lens,src,dst,block", [
    ([1, 0], [0], [1], 16), ([16, 0], [0], [1], 16), ([0, 0], [0], [1], 16),
    ([33, 0, 48, 0, 0, 0], [0, 0, 2, 2], [5, 1, 3, 4], 16), ([700, 650, 0, 0, 0, 0, 0], [1, 0, 1, 1, 0], [2, 3, 4, 5, 6], 4),
])
def test_fork_release_compact(dev, lens, src, dst, block) -> None:
    g = Both(dev, len(lens), max(1, -(-max(lens) // block)) + 2, sum(-(-n // block) for n in lens) + len(dst), block)
    g.reserve(lens)
    g.fork(src, dst)
    g.check()
    g.release(np.isin(np.arange(len(lens)), src[:1]) & (g.lens > 0))  # the source leaves before its forks
    g.check()
    g.compact()
    g.check()
    g.release(g.lens > 0)
    g.check()
    assert g.top == g.refs.shape[0]


def test_random_histories(dev) -> None:
    rng = np.random.default_rng(7)
    for seed in range(6):
        batch, block, n_pages = int(rng.integers(3, 40)), int(rng.choice([1, 4, 16])), int(rng.integers(100, 5000))
        width = max(4, n_pages // 8)
        g = Both(dev, batch, width, n_pages, block, seed=seed)
        for _ in range(25):
            what = rng.integers(5)
            empty, full = np.flatnonzero(g.lens == 0), np.flatnonzero(g.lens > 0)
            if what <= 1:
                new = rng.integers(0, max(2, width * block // 3), batch)
                new = np.minimum(new, width * block - g.lens) * (rng.random(batch) < 0.4)
                need = sum(-(-int(a + b) // block) - -(-int(a) // block) for a, b in zip(g.lens, new))
                if need <= g.top:
                    g.reserve(new)
            elif what == 2 and len(empty) and len(full):
                n = int(rng.integers(1, len(empty) + 1))
                src, dst = rng.choice(full, n), rng.permutation(empty)[:n]
                if sum(g.lens[s] % block > 0 for s in src) <= g.top:
                    g.fork(src, dst)
            elif what == 3:
                g.release((rng.random(batch) < 0.4) & (g.lens > 0))
            else:
                g.compact()
            g.check()


def test_many_forks_of_one_and_their_release(dev) -> None:
    """More than a workgroup's threads of forks; all of them leave at once, holders before and behind."""
    n = 2500
    g = Both(dev, n + 1, 40, 40 + n, 16)
    g.reserve([16 * 37 + 5] + [0] * n)
    g.fork([0] * n, list(range(1, n + 1)))
    g.check()
    rng = np.random.default_rng(0)
    g.release(rng.random(n + 1) < 0.7)
    g.check()
    g.release(g.lens > 0)
    g.check()


def test_refusals_change_nothing(dev) -> None:
    from saint_kv._lib import SKV_STATUS_BADARG as BAD, SKV_STATUS_NOSPC as NOSPC

    g = Both(dev, 6, 8, 12, 16)
    g.reserve([40, 33, 0, 0, 0, 16])
    g.fork([0], [6], BAD)
    g.fork([-1], [2], BAD)
    g.fork([0, 1], [2, 2], BAD)     # twice the same
    g.fork([0, 1], [2, 5], BAD)     # not empty
    g.check()
    g.fork([0, 5, 0, 1], [2, 3, 4, 5], BAD)
    g.reserve([16 * 3, 0, 0, 0, 0, 0])  # two pages are left
    assert g.top == 2
    g.fork([0, 0, 1], [2, 3, 4], NOSPC)
    g.check()
    g.d["bt"][1, 2] = 99            # the page to be copied is none
    g.fork([1], [2], BAD)
    g.d["bt"][1, 2] = int(g.bt[1, 2])
    g.check()
    g.fork([0, 1], [2, 3])
    g.check()
    # a page released more often than it is held: refused, counts as before
    g.d["refs"].zero_()
    g.release([1, 0, 1, 0, 0, 0], BAD)
    assert not g.d["refs"].any()
    g.d["refs"].copy_(torch.as_tensor(g.refs))
    g.check()
    g.release([1, 1, 1, 1, 0, 1])
    g.check()


def test_a_free_list_past_its_end_is_refused(dev) -> None:
    from saint_kv._lib import SKV_STATUS_STACK

    g = Both(dev, 2, 4, 8, 16)
    g.reserve([40, 0])
    g.fork([0], [1])
    g.d["top"].fill_(8)
    g.release([1, 1], SKV_STATUS_STACK)
    g.d["top"].fill_(g.top)
    g.check()


def test_a_free_list_of_pages_that_are_none_is_refused(dev) -> None:
    """A fork that would pop one writes nothing; one that needs no page goes on."""
    from saint_kv._lib import SKV_STATUS_STACK

    g = Both(dev, 4, 4, 8, 16)
    g.reserve([40, 32, 0, 0])
    for bad in (-1, 8, 2 ** 31 - 1):
        g.d["stack"][g.top - 1] = bad
        g.fork([1, 0], [2, 3], SKV_STATUS_STACK)
        g.d["stack"][g.top - 1] = int(g.stack[g.top - 1])
        g.check()
    g.d["stack"][g.top - 1] = 8
    g.fork([1], [2])
    g.d["stack"][g.top - 1] = int(g.stack[g.top - 1])
    g.check()


def test_copy_slots(dev) -> None:
    from saint_kv import ops

    g = torch.Generator(device=dev).manual_seed(0)
    shapes = [((7,), torch.int32), ((7, 3), torch.int16), ((7, 128, 64), torch.bfloat16), ((7, 3, 576), torch.float32),
              ((7, 5), torch.uint8)] + [((7, 40 * i + 8), torch.bfloat16) for i in range(40)]
    arrays = [torch.randint(-100, 100, s, generator=g, device=dev).to(t) for s, t in shapes]
    want = [a.clone() for a in arrays]
    src, dst = [0, 0, 5, 9, -1, 2], [1, 6, 3, 4, 4, 8]  # indices outside the slots copy nothing
    for w in want:
        for s, d in zip(src[:3], dst[:3]):
            w[d] = w[s]
    i32 = dict(dtype=torch.int32, device=dev)
    ops.copy_slots(arrays, torch.tensor(src, **i32), torch.tensor(dst, **i32))
    assert all(torch.equal(a, w) for a, w in zip(arrays, want))
    with pytest.raises(ValueError):
        ops.copy_slots([arrays[0], arrays[1][:4]], torch.tensor(src, **i32), torch.tensor(dst, **i32))
    with pytest.raises(ValueError):
        ops.copy_slots([arrays[2][:, ::2]], torch.tensor(src, **i32), torch.tensor(dst, **i32))


def test_captured_fork_and_release_replay(dev) -> None:
    """The same fork and release replayed over tables that eager calls change in between."""
    g = Both(dev, 4, 8, 30, 16)
    g.reserve([37, 50, 0, 0])
    d = g.d
    src, dst = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 1], [2, 3]))
    mask = torch.tensor([0, 0, 1, 1], dtype=torch.uint8, device=dev)

    def work():
        g.ops.fork(d["stack"], d["top"], d["refs"], d["bt"], d["lens"], src, dst, 16, g.dpools, d["status"])
        g.ops.release(d["stack"], d["top"], d["bt"], d["lens"], mask, 16, d["status"], refs=d["refs"])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for n in range(3):
        graph.replay()
        g.top = ora.fork(g.stack, g.top, g.refs, g.bt, g.lens, [0, 1], [2, 3], 16, g.pools)
        g.top = ora.release(g.stack, g.top, g.refs, g.bt, g.lens, mask.cpu().numpy(), 16)
        g.check()
        g.reserve([5, 3, 0, 0])
        g.check()


# --------------------------------------------------------------------------- the decode cache
def _decode_cache(dev, batch=5, **kw):
    from saint_kv import DecodeCache, LayerSpec

    layers = [LayerSpec("csa", m=4, top_k=8), LayerSpec("hca", m=8), LayerSpec("csa", m=4, top_k=8, indexer=False),
              LayerSpec("swa")]
    return DecodeCache(layers, batch, 512, latent=64, c_indexer=32, window=16, block_size=4, device=dev, **kw)


def _rows(cache, g, b, t):
    out = []
    for i in range(len(cache.layers)):
        out.append({n: torch.randn(b, t, x.shape[-1], generator=g, device=cache.device).to(torch.bfloat16)
                    for n, x in cache.inputs[i].items()})
    return out


def test_decode_cache_forks_continue_as_their_source(dev) -> None:
    """A sequence forked twice: fed what the source is fed, both give what it gives, also after the source has
    left and the pages have been compacted; fed other tokens, they give what a cache of their own gives."""
    cache, alone = _decode_cache(dev), _decode_cache(dev, page_order_seed=3)
    g = torch.Generator(device=dev).manual_seed(0)
    lens = np.array([203, 0, 77, 0, 0])
    data = _rows(cache, g, 5, 203)
    cache.prefill(lens, data=data)
    alone.prefill(np.array([203, 203, 77, 203, 0]), data=[{n: x[[0, 0, 2, 0, 4]] for n, x in d.items()} for d in data])
    cache.fork([0, 0], [1, 3])
    live = [0, 1, 2, 3]

    def same():
        for i, spec in enumerate(cache.layers):
            assert torch.equal(cache.out_window[i][live], alone.out_window[i][live])
            if spec.kind == "csa":
                assert torch.equal(cache.topk_idx[i][live], alone.topk_idx[i][live])
                assert torch.equal(cache.out_entries[i][live], alone.out_entries[i][live])
            elif spec.kind == "hca":
                for b in live:
                    n = int(cache.host_lens[b]) // spec.m
                    assert torch.equal(cache.out_entries[i][b, :n], alone.out_entries[i][b, :n])

    def step(together):
        for i, row in enumerate(_rows(cache, g, 5, 1)):
            for n, x in row.items():
                x = x[:, 0]
                if together:
                    x = x[[0, 0, 2, 0, 4]]
                cache.inputs[i][n].copy_(x)
                alone.inputs[i][n].copy_(x)
            if cache.scores[i] is not None:
                s = torch.randn(cache.scores[i].shape, generator=g, device=dev)
                cache.scores[i].copy_(s)
                alone.scores[i].copy_(s)
        cache.step()
        alone.step()
        cache.check_status()
        same()

    for _ in range(6):
        step(True)
    for _ in range(7):
        step(False)
    cache.release(np.array([1, 0, 0, 0, 1], dtype=bool))
    alone.release(np.array([1, 0, 0, 0, 1], dtype=bool))
    cache.compact()
    live[:] = [1, 2, 3]
    for _ in range(9):
        step(False)
    cache.release(np.array([1, 0, 0, 0, 0], dtype=bool))  # a step gives every slot a token, the empty ones too
    cache.fork(1, 0)
    cache.release(np.array([1, 1, 1, 1, 1], dtype=bool))
    for grp in cache.groups:
        assert int(grp.free_top) == grp.n_pages and not grp.refs.any()


def test_decode_cache_fork_refusals_leave_it_as_it_was(dev) -> None:
    cache = _decode_cache(dev, pages_per_group={4: 30, 8: 8})
    g = torch.Generator(device=dev).manual_seed(1)
    # 101 tokens: 25 entries of m = 4 (7 pages), 12 of m = 8 (3 whole pages); 110: 13 entries, 4 pages
    data = _rows(cache, g, 5, 120)
    cache.prefill(np.array([101, 110, 0, 0, 0]), data=data)
    before = [(grp.block_table.clone(), grp.free_top.clone(), grp.n_entries.clone()) for grp in cache.groups]
    with pytest.raises(RuntimeError, match="refused"):
        cache.fork([1, 1], [2, 3])  # m = 8 has one page left
    for grp, (bt, top, ne) in zip(cache.groups, before):
        assert torch.equal(grp.block_table, bt) and torch.equal(grp.free_top, top) and torch.equal(grp.n_entries, ne)
        assert not grp.refs.any()
    assert cache.host_lens.tolist() == [101, 110, 0, 0, 0] and cache.tok_lens.tolist() == [101, 110, 0, 0, 0]
    for bad in (([0], [1]), ([0, 0], [2])):
        with pytest.raises((RuntimeError, ValueError)):
            cache.fork(*bad)
    cache.fork(0, 2)
    assert cache.host_lens.tolist() == [101, 110, 101, 0, 0]
    cache.release(np.array([1, 1, 1, 0, 0], dtype=bool))


def test_a_window_only_cache_forks(dev) -> None:
    from saint_kv import DecodeCache, LayerSpec

    cache = DecodeCache([LayerSpec("swa")], 3, 64, latent=64, window=8, device=dev)
    cache.prefill(np.array([11, 0, 5]), data=[{"kv": torch.randn(3, 11, 64, device=dev).to(torch.bfloat16)}])
    cache.fork(0, 1)
    assert torch.equal(cache.ring[0][0], cache.ring[0][1]) and cache.tok_lens.tolist() == [11, 11, 5]
