"""Random histories of the 4-bit cache against plain lists of what each sequence should hold, and
its attention over random shapes against the formula."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_fp4_attention import check, make

from oracle import fp4_cache as ora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(6))
def test_what_sequences_hold(dev, seed) -> None:
    """Ragged and uniform reservations, forks, releases, compactions in any order: every layer reads back
    its tokens, in 64 bits from the values that went in, and no page is lost or held twice without a count."""
    from saint_kv import Fp4TokenCache, ops

    rng = np.random.default_rng(seed)
    layers, batch, kv, dim, block = 2, int(rng.integers(3, 9)), int(rng.integers(1, 4)), int(rng.choice([32, 64, 96, 128])), 16
    max_len = int(rng.integers(40, 300))
    pages = int(batch * -(-max_len // block) * rng.uniform(0.5, 1.0))
    cache = Fp4TokenCache(layers, batch, max_len, kv, dim, block_size=block, n_pages=pages, device=dev)
    held = [[[] for _ in range(batch)] for _ in range(layers)]  # per layer and sequence: (k, v) of every token
    lens = np.zeros(batch, dtype=np.int64)
    for _ in range(40):
        what = rng.choice(["reserve", "reserve", "uniform", "fork", "release", "compact"])
        if what in ("reserve", "uniform"):
            if what == "uniform":
                n = np.full(batch, int(rng.integers(1, 4)))
            else:
                n = (rng.integers(0, max_len // 2, batch) * (rng.random(batch) < 0.5)).astype(np.int64)
            n = np.minimum(n, max_len - lens) if what == "reserve" else n
            try:
                cache.reserve(int(n[0]) if what == "uniform" else n)
            except RuntimeError as e:
                assert "overflow" in str(e) or "out of pages" in str(e)
                continue
            lens = lens + n
            t = int(n.max()) + (int(rng.integers(0, 3)) if what == "reserve" else 0)
            for i in range(layers):
                x = rng.standard_normal((2, batch, max(t, 1), kv, dim))
                k, v = (torch.as_tensor(y, device=dev).to(torch.bfloat16) for y in x)
                cache.append(i, k, v)
                kh, vh = k.double().cpu().numpy(), v.double().cpu().numpy()
                for b in range(batch):
                    held[i][b] += [(kh[b, j], vh[b, j]) for j in range(int(n[b]))]
        elif what == "fork":
            full, empty = np.flatnonzero(lens > 0), np.flatnonzero(lens == 0)
            if not len(full) or not len(empty):
                continue
            src = rng.choice(full, int(rng.integers(1, len(empty) + 1)))
            dst = rng.permutation(empty)[:len(src)]
            try:
                cache.fork(src, dst)
            except RuntimeError as e:
                assert "out of pages" in str(e)
                continue
            lens[dst] = lens[src]
            for h in held:
                for s, d in zip(src, dst):
                    h[d] = list(h[s])
        elif what == "release":
            mask = (rng.random(batch) < 0.4) & (lens > 0)
            cache.release(mask)
            lens[mask] = 0
            for h in held:
                for b in np.flatnonzero(mask):
                    h[b] = []
        else:
            live, _ = cache.compact()
            assert live == cache.n_pages - cache.host_free
        cache.check_status()
        assert cache.host_lens.tolist() == lens.tolist() == cache.seq_lens.tolist()
        table, refs = cache.block_table.cpu().numpy(), cache.refs.cpu().numpy()
        owned = np.concatenate([table[b, :-(-int(lens[b]) // block)] for b in range(batch)] + [np.zeros(0, np.int64)])
        count = np.bincount(owned.astype(np.int64), minlength=pages)
        assert np.array_equal(refs, np.maximum(count - 1, 0)) and cache.host_free == int(cache.free_top) == int((count == 0).sum())
        top = max(1, int(lens.max()))
        for i in range(layers):
            out = [torch.zeros(batch, top, kv, dim, dtype=torch.bfloat16, device=dev) for _ in range(2)]
            ops.fp4_gather(cache.pool[i], cache.block_table, cache.seq_lens, *out, cache.seq_lens)
            for c in range(2):
                got = out[c].double().cpu().numpy()
                for b in range(batch):
                    if lens[b]:
                        x = np.stack([tok[c] for tok in held[i][b]])
                        codes, scales = ora.quantize(x.reshape(-1, dim))
                        assert np.array_equal(got[b, :lens[b]], ora.dequantize(codes, scales).reshape(x.shape)), (i, c, b)


@pytest.mark.parametrize("seed", range(40))
def test_random_shapes(dev, seed) -> None:
    from saint_kv import fp4_attention

    rng = np.random.default_rng(1000 + seed)
    batch, kv, block = int(rng.integers(1, 7)), int(rng.choice([1, 1, 2, 3, 8])), 16 * int(rng.integers(1, 6))
    dim, group = 32 * int(rng.integers(1, 17)), int(rng.choice([1, 2, 3, 7, 16, 40]))
    t = int(rng.choice([1, 1, 2, 5, 23, 70]))
    if t * group > 200:
        t = max(1, 200 // group)
    lens = np.round(np.exp(rng.uniform(0, np.log(900 if t * group < 70 else 300), batch))).astype(np.int64) - (rng.random(batch) < 0.1)
    pool, bt, lens_t = make(dev, lens, block, kv, dim, seed=seed, spare=int(rng.integers(0, 3)))
    if rng.random() < 0.3:
        bt[int(rng.integers(batch)), int(rng.integers(bt.shape[1]))] = -1
    q = torch.as_tensor(rng.standard_normal((batch, t, kv * group, dim)), device=dev).to(torch.bfloat16)
    kw = {}
    if rng.random() < 0.4:
        kw["window"] = int(np.round(np.exp(rng.uniform(0, np.log(400)))))
    if rng.random() < 0.4:
        kw["sink"] = torch.as_tensor(rng.standard_normal(kv * group), device=dev).float()
    if rng.random() < 0.4:
        kw["softcap"] = float(np.exp(rng.uniform(np.log(0.5), np.log(1e6))))
    if rng.random() < 0.3:
        kw["scale"] = float(np.exp(rng.uniform(np.log(0.001), np.log(0.3))))
    n_new = None
    if rng.random() < 0.4:
        n_new = rng.integers(0, t + 1, batch).astype(np.int32)
    given = dict(kw, n_new=None if n_new is None else torch.as_tensor(n_new, device=dev))
    first = None
    for extra in (dict(), dict(splits=int(rng.integers(1, 6))), dict(max_len=int(rng.integers(1, 1000)))):
        got = fp4_attention(q, pool, bt, lens_t, **given, **extra)
        check(got, q, pool, bt, lens_t, **dict(kw, **({} if n_new is None else {"n_new": n_new})))
        first = got if first is None else first
    assert torch.equal(first, fp4_attention(q, pool, bt, lens_t, **given))
