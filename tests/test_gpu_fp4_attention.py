"""Attention over the 4-bit pages against the formula in 64 bits on the very bytes of the pages.

Tolerance, per output: the weights are rounded to bf16 for the product with the values (half a step,
2^-8 of each term, so 2^-8 of A = sum w |v| / (sum w + sink)), the output once (2^-8 of it); the
rest is fp32: a score's products and sums err by less than D 2^-24 sum |q k| scale, with the exponential
a few 2^-24 of its argument's size more, together below 2^-2 of a bf16 half step for the scores here
(|s| < 60): 2^-8 |want| + 1.25 * 2^-8 A.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp4_cache as ora

pytestmark = pytest.mark.gpu


def make(dev, lens, block, heads, dim, seed=0, spare=1):
    """Pages of normally distributed tokens behind stale ones (a NaN block among them), a shuffled table."""
    from saint_kv import ops

    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, dtype=np.int32)
    pages = -(-lens // block)
    n_pages = int(pages.sum()) + 2
    pool = ops.fp4_pool(n_pages, block, heads, dim, dev)
    pool.fill_(0xFF)  # stale bytes: every scale byte is NaN's
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


def check(got, q, pool, bt, lens, **kw):
    """Elementwise, within the bound of the module's docstring."""
    qn, pn, btn, ln = q.cpu().double().numpy(), pool.cpu().numpy(), bt.cpu().numpy(), lens.cpu().numpy()
    kw = {n: x.cpu().numpy() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    want = ora.attention(qn, pn, btn, ln, **kw)
    mag = pn.copy()
    p = ora.Pages(mag)
    half = p.block * p.dim // 2
    p.flat[:, :, half:2 * half] &= 0x77  # |v|: the signs of the values' codes cleared
    a = ora.attention(qn, mag, btn, ln, **kw)
    g = got.detach().cpu().double().numpy().reshape(want.shape)
    assert np.array_equal(np.isnan(g), np.isnan(want))
    off = np.abs(g - want) - (2.0 ** -8 * np.abs(want) + 1.25 * 2.0 ** -8 * a)
    off[np.isnan(want)] = -1
    assert (off <= 0).all(), f"worst {off.max()} at {np.unravel_index(off.argmax(), off.shape)}"


CASES = [
    # lens, T, H, Hkv, D, block, window, sink, softcap
    ([1], 1, 1, 1, 32, 16, None, False, None),
    ([333], 1, 16, 2, 128, 16, None, False, None),
    ([0, 1, 15, 16, 17, 31, 32, 33], 1, 4, 1, 64, 16, None, True, None),
    ([64, 65, 127, 500], 1, 6, 2, 96, 64, None, False, 20.0),
    ([200, 3, 77], 4, 8, 4, 128, 32, None, True, None),
    ([50, 2, 0, 130], 7, 5, 5, 160, 16, None, False, None),
    ([300, 129, 40], 1, 64, 1, 512, 16, 128, True, 30.0),
    ([300, 20], 3, 24, 1, 256, 48, 33, False, None),
    ([400, 90], 40, 16, 2, 64, 64, None, False, None),
    ([260, 33], 33, 3, 1, 128, 16, 50, True, None),
    ([150, 131], 130, 8, 2, 128, 128, None, False, None),
    ([90, 70], 70, 2, 2, 512, 16, 1, False, None),
    ([700], 65, 17, 1, 32, 16, None, True, 5.0),
    ([128, 513], 16, 32, 2, 192, 64, None, False, None),
    ([1000, 999, 5], 1, 12, 3, 224, 16, 700, False, None),
]


@pytest.mark.parametrize("lens,t,heads,kv,dim,block,window,sink,softcap", CASES)
def test_attention(dev, lens, t, heads, kv, dim, block, window, sink, softcap) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens_t = make(dev, lens, block, kv, dim, seed=dim + t)
    g = torch.Generator(device=dev).manual_seed(t)
    q = torch.randn(len(lens), t, heads, dim, generator=g, device=dev).to(torch.bfloat16)
    kw = dict(window=window, softcap=softcap, sink=torch.randn(heads, generator=g, device=dev) if sink else None)
    for splits in (0, 1, 3):
        got = fp4_attention(q, pool, bt, lens_t, splits=splits, **kw)
        assert got.dtype == torch.bfloat16 and got.shape == q.shape
        check(got, q, pool, bt, lens_t, **kw)
    if t == 1:
        assert torch.equal(fp4_attention(q[:, 0], pool, bt, lens_t, splits=3, **kw), got[:, 0])


@pytest.mark.parametrize("t,heads,kv,dim,max_len", [(1, 8, 1, 128, 0), (1, 64, 1, 64, 5000), (2, 8, 4, 128, 100),
                                                    (100, 4, 1, 128, 5000), (1, 16, 1, 512, 5000)])
def test_long_sequences_over_several_workgroups(dev, t, heads, kv, dim, max_len) -> None:
    """Splits chosen by the library, the lengths ragged; a bound that is too low is still right."""
    from saint_kv import fp4_attention

    lens = [4800, 100, 0, 2049]
    pool, bt, lens_t = make(dev, lens, 64, kv, dim, seed=5, spare=40)
    q = torch.randn(4, t, heads, dim, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    got = fp4_attention(q, pool, bt, lens_t, max_len=max_len)
    check(got, q, pool, bt, lens_t)
    assert torch.equal(got, fp4_attention(q, pool, bt, lens_t, max_len=max_len))  # no order that changes


@pytest.mark.parametrize("t,heads", [(1, 2), (1, 40), (20, 8)])
def test_large_scores_and_scale(dev, t, heads) -> None:
    """Scores of some hundreds: the running maximum moves often, single keys take all the weight."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [777, 64], 16, 2, 128, seed=9)
    g = torch.Generator(device=dev).manual_seed(2)
    q = (torch.randn(2, t, heads, 128, generator=g, device=dev) * 8).to(torch.bfloat16)
    sink = torch.full((heads,), -1e30, device=dev)
    # |s| is up to about 60 here, as the tolerance assumes
    check(fp4_attention(q, pool, bt, lens, sink=sink), q, pool, bt, lens, sink=sink)
    check(fp4_attention(q, pool, bt, lens, scale=0.002), q, pool, bt, lens, scale=0.002)
    sink = torch.full((heads,), 200.0, device=dev)
    assert (fp4_attention(q, pool, bt, lens, sink=sink).float().abs() < 1e-30).all()


@pytest.mark.parametrize("t,heads,dim", [(1, 4, 128), (1, 64, 128), (40, 8, 64), (5, 4, 512)])
def test_nan_blocks_reach_only_the_tokens_that_see_them(dev, t, heads, dim) -> None:
    from saint_kv import fp4_attention, ops

    lens = [300, 300, 200]
    pool, bt, lens_t = make(dev, lens, 16, 1, dim, seed=3)
    # a NaN key in sequence 0 at position 296, a NaN value in sequence 1 at position 100
    for b, pos, which in ((0, 296, 0), (1, 100, 1)):
        x = torch.randn(3, 1, 1, dim, device=dev).to(torch.bfloat16)
        y = x.clone()
        (x if which == 0 else y)[b, 0, 0, dim - 1] = float("nan")
        at, n = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
        at[b], n[b] = pos + 1, 1
        ops.fp4_quant_append(pool, bt, at, x, y, n)
    q = torch.randn(3, t, heads, dim, device=dev).to(torch.bfloat16)
    got = fp4_attention(q, pool, bt, lens_t)
    check(got, q, pool, bt, lens_t)
    got = fp4_attention(q, pool, bt, lens_t, window=60)  # sequence 1 no longer sees its own
    check(got, q, pool, bt, lens_t, window=60)
    assert not torch.isnan(got[1:]).any()


@pytest.mark.parametrize("t,heads", [(1, 4), (1, 48), (30, 8)])
def test_unmapped_pages_are_not_seen(dev, t, heads) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [250, 100, 60], 16, 1, 64, seed=4)
    bt[0, 3], bt[0, 9] = -1, pool.shape[0]
    bt[1, :] = -7
    q = torch.randn(3, t, heads, 64, device=dev).to(torch.bfloat16)
    got = fp4_attention(q, pool, bt, lens)
    check(got, q, pool, bt, lens)
    assert (got[1] == 0).all()


def test_lengths_past_the_table_and_below_zero(dev) -> None:
    """A length that the table cannot hold sees what it holds; a negative one sees nothing."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [64, 64], 16, 1, 64, spare=0)
    q = torch.randn(2, 1, 2, 64, device=dev).to(torch.bfloat16)
    want = fp4_attention(q, pool, bt, lens)
    got = fp4_attention(q, pool, bt, torch.tensor([1 << 30, -5], dtype=torch.int32, device=dev))
    assert torch.equal(got[0], want[0]) and (got[1] == 0).all()


def test_strided_queries_and_given_buffers(dev) -> None:
    from saint_kv import fp4_attention
    from saint_kv.fp4 import fp4_attention_workspace

    pool, bt, lens = make(dev, [900, 450], 64, 2, 128, seed=6)
    q = torch.randn(2, 8, 3, 128, device=dev).to(torch.bfloat16)  # [B, H, T, D], as a forward holds it
    got = fp4_attention(q.transpose(1, 2), pool, bt, lens, splits=4)
    assert torch.equal(got, fp4_attention(q.transpose(1, 2).contiguous(), pool, bt, lens, splits=4))
    need = fp4_attention_workspace(q.transpose(1, 2), pool, bt, splits=4)
    out = torch.full_like(got, 3.0)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    assert fp4_attention(q.transpose(1, 2), pool, bt, lens, splits=4, out=out, workspace=ws) is out
    assert torch.equal(out, got)
    if need > 16:
        with pytest.raises(ValueError, match="workspace"):
            fp4_attention(q.transpose(1, 2), pool, bt, lens, splits=4, workspace=ws[:need - 16])


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
    q = torch.randn(2, 1, heads, dim, device=dev).to(torch.bfloat16)
    got = fp4_attention(q, pool, bt, lens)
    ids = torch.unique(bt).long()
    small = torch.searchsorted(ids, bt.long()).to(torch.int32)
    check(got, q, pool[ids], small, lens)


def test_refusals(dev) -> None:
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [40, 40], 16, 2, 64)
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device=dev)
    ok = dict(q=q, pool=pool, block_table=bt, seq_lens=lens)
    for bad in (dict(q=q.float()), dict(q=q[:1]), dict(q=q[:, :, :3]), dict(q=q[..., :32]), dict(q=q[:, :0]),
                dict(seq_lens=lens.long()), dict(seq_lens=lens[:1]), dict(window=0), dict(softcap=0.0), dict(softcap=-1.0),
                dict(scale=0.0), dict(scale=float("nan")), dict(sink=torch.zeros(3, device=dev)),
                dict(sink=torch.zeros(4, dtype=torch.bfloat16, device=dev)), dict(out=torch.zeros_like(q.float())),
                dict(out=torch.zeros_like(q)[:1]), dict(max_len=-1), dict(splits=-1),
                dict(q=torch.zeros(2, 1, 4, 72, dtype=torch.bfloat16, device=dev)[..., 4:68])):
        with pytest.raises(ValueError):
            fp4_attention(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="CPU"):
        fp4_attention(**{**ok, "seq_lens": lens.cpu()})


def test_captured_attention_replays(dev) -> None:
    """Two graphs of their own workspaces, replayed in turn over lengths that eager work changes."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [2000, 700], 64, 1, 128, seed=8)
    q = torch.zeros(2, 1, 8, 128, dtype=torch.bfloat16, device=dev)
    q2 = torch.zeros(2, 9, 8, 128, dtype=torch.bfloat16, device=dev)
    fp4_attention(q, pool, bt, lens)
    fp4_attention(q2, pool, bt, lens)
    torch.cuda.synchronize()
    graphs = []
    for x in (q, q2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp4_attention(x, pool, bt, lens)
        graphs.append((graph, x, y))
    for n in range(4):
        lens.copy_(torch.tensor([2000 - 700 * (n % 2), 700 - 90 * n], dtype=torch.int32))
        for graph, x, _ in graphs:
            x.copy_(torch.randn(x.shape, device=dev))
            graph.replay()
        torch.cuda.synchronize()
        for _, x, y in graphs:
            assert torch.equal(y, fp4_attention(x, pool, bt, lens))
