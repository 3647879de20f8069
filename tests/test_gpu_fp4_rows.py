"""Tokens into the 4-bit pages and back: every byte of the pages against the oracle, every
value bit for bit (both directions are exact), over heads, dims, pages, strides and counts."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp4_cache as ora

pytestmark = pytest.mark.gpu


def _cache(dev, lens, block, heads, dim, seed=0, fill=0xA5):
    """A pool of stale bytes, a shuffled block table over it (one page left unmapped nowhere), lengths."""
    from saint_kv import ops

    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, dtype=np.int32)
    width = max(1, int(-(-lens.max() // block))) + 1
    pages = -(-lens // block)
    n_pages = int(pages.sum()) + 2
    pool = ops.fp4_pool(n_pages, block, heads, dim, dev)
    pool.fill_(fill)
    order, at = rng.permutation(n_pages).astype(np.int32), 0
    bt = np.full((len(lens), width), -1, dtype=np.int32)
    for b, p in enumerate(pages):
        bt[b, :p] = order[at:at + p]
        at += p
    return pool, torch.as_tensor(bt, device=dev), torch.as_tensor(lens, device=dev)


def _values(g, *shape, dev, dtype):
    x = torch.randn(*shape, generator=g, device=dev) * 2.0 ** torch.randint(-12, 12, shape[:-1], generator=g,
                                                                           device=dev)[..., None]
    return x.to(dtype)


def _np(t):
    return t.detach().cpu().to(torch.float64).numpy()


@pytest.mark.parametrize("lens,n_new,block,heads,dim,dtype", [
    ([1], [1], 16, 1, 32, torch.bfloat16), ([17, 40, 64], [1, 1, 1], 16, 2, 64, torch.bfloat16),
    ([33, 5, 0, 100], [33, 2, 0, 51], 16, 3, 96, torch.bfloat16), ([130, 64], [130, 64], 64, 8, 128, torch.float32),
    ([90, 31], [7, 31], 32, 1, 512, torch.bfloat16), ([300, 299, 1], [255, 1, 1], 48, 2, 160, torch.float32),
    ([20, 20], [0, 0], 16, 1, 256, torch.bfloat16),
])
def test_append_and_gather(dev, lens, n_new, block, heads, dim, dtype) -> None:
    from saint_kv import ops

    g = torch.Generator(device=dev).manual_seed(len(lens) + dim)
    pool, bt, lens_t = _cache(dev, lens, block, heads, dim)
    t = max(max(n_new), 1) + 2  # tokens of k and v behind the new ones are not read
    k, v = (_values(g, len(lens), t, heads, dim, dev=dev, dtype=dtype) for _ in range(2))
    k[:, :, 0, :32] *= 0  # a block of zeros, of both signs
    k[:, :, 0, 3] = -0.0
    want = pool.cpu().numpy().copy()
    ora.append(want, bt.cpu().numpy(), np.asarray(lens), _np(k), _np(v), np.asarray(n_new))
    n_t = torch.as_tensor(np.asarray(n_new, dtype=np.int32), device=dev)
    ops.fp4_quant_append(pool, bt, lens_t, k, v, n_t)
    assert np.array_equal(pool.cpu().numpy(), want)
    shape = (len(lens), t, heads, dim)
    out = [torch.full(shape, 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    ops.fp4_gather(pool, bt, lens_t, *out, n_t)
    for b, n in enumerate(n_new):
        kk, vv, _ = ora.rows(want, bt.cpu().numpy(), b, range(lens[b] - n, lens[b]))
        for got, exp in zip(out, (kk, vv)):
            assert np.array_equal(_np(got[b, :n]), exp) and (got[b, n:] == 7).all()


def test_uniform_counts_strided_rows_and_heads(dev) -> None:
    """k and v as slices of one fused projection, heads before tokens; out into slices too."""
    from saint_kv import ops

    g = torch.Generator(device=dev).manual_seed(1)
    heads, dim, t = 4, 64, 9
    pool, bt, lens = _cache(dev, [9, 30], 16, heads, dim)
    fused = torch.randn(2, heads, t, 3 * dim, generator=g, device=dev).to(torch.bfloat16)
    k, v = fused[..., dim:2 * dim].transpose(1, 2), fused[..., 2 * dim:].transpose(1, 2)
    ops.fp4_quant_append(pool, bt, lens, k, v, t)
    want = torch.zeros_like(pool)
    want.fill_(0xA5)
    ops.fp4_quant_append(want, bt, lens, k.contiguous(), v.contiguous(), t)
    assert torch.equal(pool, want)
    out = torch.zeros(2, t, heads, 2, dim, dtype=torch.bfloat16, device=dev)
    ops.fp4_gather(pool, bt, lens, out[..., 0, :], out[..., 1, :], t)
    a, b = torch.zeros(2, t, heads, dim, dtype=torch.bfloat16, device=dev), torch.zeros(2, t, heads, dim,
                                                                                     dtype=torch.bfloat16, device=dev)
    ops.fp4_gather(pool, bt, lens, a, b, t)
    assert torch.equal(out[..., 0, :], a) and torch.equal(out[..., 1, :], b)


def test_every_bf16_value(dev) -> None:
    """All 2^16 bf16 patterns, each the largest of its block, and each beside a 6: codes and scales."""
    from saint_kv import ops

    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    k = torch.zeros(1, 4096, 16, 32, dtype=torch.bfloat16)
    k[..., 5] = every.view(1, 4096, 16)
    v = k.clone()
    v[..., 9] = -6.0
    pool, bt, lens = _cache(dev, [4096], 64, 16, 32)
    want = pool.cpu().numpy().copy()
    ora.append(want, bt.cpu().numpy(), np.array([4096]), _np(k), _np(v), np.array([4096]))
    ops.fp4_quant_append(pool, bt, lens, k.to(dev), v.to(dev), 4096)
    assert np.array_equal(pool.cpu().numpy(), want)
    out_k, out_v = (torch.zeros(1, 4096, 16, 32, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ops.fp4_gather(pool, bt, lens, out_k, out_v, 4096)
    kk, vv, _ = ora.rows(want, bt.cpu().numpy(), 0, range(4096))
    assert np.array_equal(_np(out_k[0]), kk, equal_nan=True) and np.array_equal(_np(out_v[0]), vv, equal_nan=True)


def test_all_code_bytes_under_all_scales(dev) -> None:
    from saint_kv import ops

    heads, dim, n = 8, 512, 64
    pool, bt, lens = _cache(dev, [n], 64, heads, dim)
    p = ora.Pages(pool.cpu().numpy())
    page = int(bt[0, 0])
    half = 64 * dim // 2
    p.flat[page, :, :2 * half] = np.arange(2 * half) % 256
    p.flat[page, :, 2 * half:] = (np.arange(64 * 32)[None] + 13 * np.arange(heads)[:, None]) % 253
    pool.copy_(torch.as_tensor(p.pool))
    out_k, out_v = (torch.zeros(1, n, heads, dim, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ops.fp4_gather(pool, bt, lens, out_k, out_v, n)
    kk, vv, _ = ora.rows(p.pool, bt.cpu().numpy(), 0, range(n))
    assert np.array_equal(_np(out_k[0]), kk) and np.array_equal(_np(out_v[0]), vv)


def test_counts_that_are_no_append_and_unmapped_pages(dev) -> None:
    """More new tokens than the length, negative counts and lengths, pages outside the pool: nothing is written
    there, zeros are read; the other sequences are not touched by it."""
    from saint_kv import ops

    heads, dim = 1, 64
    pool, bt, lens = _cache(dev, [40, 40, 40, 40, 40], 16, heads, dim)
    k = torch.randn(5, 40, heads, dim, device=dev).to(torch.bfloat16)
    bt[2, 1], bt[3, 0] = -1, pool.shape[0]
    lens[4] = -3
    n = torch.tensor([41, -2, 40, 40, 1], dtype=torch.int32, device=dev)
    before = pool.clone()
    ops.fp4_quant_append(pool, bt, lens, k, k, n)
    want = before.cpu().numpy()
    kn = _np(k)
    for b, hole in ((2, range(16, 32)), (3, range(16))):
        p = ora.Pages(want)
        for pos in range(40):
            if pos not in hole:
                for kv in range(2):
                    p.write(int(bt[b, pos // 16]), pos % 16, kv, kn[b, pos])
    assert np.array_equal(pool.cpu().numpy(), want)
    out = torch.full((5, 40, heads, dim), 7.0, dtype=torch.bfloat16, device=dev)
    ops.fp4_gather(pool, bt, lens, out, torch.zeros_like(out), n)
    assert (out[[0, 1, 4]] == 7).all() and (out[2, 16:32] == 0).all() and (out[3, :16] == 0).all()
    assert not (out[2, :16] == 7).any()


def test_a_far_page_and_another_stream(dev) -> None:
    """A pool past 4 GiB, a page at its end; written on one stream, read on another that waits."""
    from saint_kv import ops

    heads, dim, block = 8, 512, 128
    n_pages = (9 << 30) // (block * heads * dim * 17 // 16 * 2)
    pool = torch.empty(n_pages, block, heads, 17 * dim // 16, dtype=torch.uint8, device=dev)
    assert pool.numel() > 1 << 32
    bt = torch.tensor([[0, n_pages - 1]], dtype=torch.int32, device=dev)
    lens = torch.tensor([block + 5], dtype=torch.int32, device=dev)
    k = torch.randn(1, block + 5, heads, dim, device=dev).to(torch.bfloat16)
    v = torch.randn(1, block + 5, heads, dim, device=dev).to(torch.bfloat16)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        ops.fp4_quant_append(pool, bt, lens, k, v, block + 5)
    torch.cuda.current_stream(dev).wait_stream(s)
    a, b = torch.zeros_like(k), torch.zeros_like(v)
    ops.fp4_gather(pool, bt, lens, a, b, block + 5)
    for got, x in ((a, k), (b, v)):
        assert np.array_equal(_np(got), ora.dequantize(*ora.quantize(_np(x))))


def test_refusals(dev) -> None:
    from saint_kv import ops

    pool, bt, lens = _cache(dev, [40, 40], 16, 2, 64)
    k = torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16, device=dev)
    ok = dict(pool=pool, block_table=bt, seq_lens=lens, k=k, v=k, n_new=8)
    for bad in (dict(k=k.half()), dict(k=k[:1]), dict(k=k[:, :, :1]), dict(k=k[..., :32]), dict(v=k.float()),
                dict(v=k[:, :7]), dict(n_new=9), dict(n_new=-1), dict(n_new=lens[:1]), dict(seq_lens=lens.long()),
                dict(block_table=bt[0]), dict(pool=pool[..., :-1]), dict(pool=pool.view(-1, 8, 4, 68)),
                dict(k=torch.zeros(2, 8, 2, 72, dtype=torch.bfloat16, device=dev)[..., 4:68]),
                dict(k=torch.zeros(2, 8, 2, 128, dtype=torch.bfloat16, device=dev)[..., ::2])):
        with pytest.raises(ValueError):
            ops.fp4_quant_append(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="CPU"):
        ops.fp4_quant_append(**{**ok, "k": k.cpu()})
    with pytest.raises(ValueError):
        ops.fp4_gather(pool, bt, lens, k.float(), k.float(), 8)


def test_a_captured_write_and_read_replays_on_new_rows(dev) -> None:
    from saint_kv import ops

    pool, bt, lens = _cache(dev, [8, 8], 16, 2, 64)
    k, v = (torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(2))
    a, b = torch.zeros_like(k), torch.zeros_like(v)

    def work():
        ops.fp4_quant_append(pool, bt, lens, k, v, 8)
        ops.fp4_gather(pool, bt, lens, a, b, 8)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for seed in range(4):
        g = torch.Generator(device=dev).manual_seed(seed)
        k.copy_(torch.randn(k.shape, generator=g, device=dev))
        v.copy_(torch.randn(k.shape, generator=g, device=dev))
        graph.replay()
        got = a.clone(), b.clone()
        torch.cuda.synchronize()
        work()
        assert torch.equal(a, got[0]) and torch.equal(b, got[1])
        assert np.array_equal(_np(a), ora.dequantize(*ora.quantize(_np(k))))
