"""The weights of the 4-bit attention's products where each wave has tiles of its own: carried as
a bf16 and the bf16 of what that leaves.

Pairs of keys have opposite values and nearly equal weights, so that an output is small beside
A = sum w |v| / sum w and an error of the weights shows: rounded to bf16 once (half a step of 2^-8, as
where the waves share their tiles) they err by 2^-10 A on average.

Bound, from the arithmetic: the output's own rounding, 2^-8 |want|; the weights', 2^-8 of what 2^-8
left, 2^-16 A; a score's products and sums, D 2^-24 sum |q k| scale <= 512 * 2^-24 * 512 * 0.7 * 0.002 = 2.2e-5,
in numerator and denominator; the sums over up to 80 keys, 80 * 2^-24 A; exp2, 2^-22 A.  With all of
them at their worst 2^-14 A.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_fp4_attention import make

from oracle import fp4_cache as ora

SCALE = 0.002


def bound(want: np.ndarray, a: np.ndarray) -> np.ndarray:
    return 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * a


def _bf16(x: np.ndarray) -> np.ndarray:
    return torch.as_tensor(x).to(torch.bfloat16).double().numpy()


def test_the_bound_tells_whole_weights_from_rounded_ones() -> None:
    """Weights with their rests keep it; without, or with the rest of the wrong sign, most outputs of few keys do not."""
    rng = np.random.default_rng(0)
    for n, dim in ((2, 64), (8, 128), (40, 512)):
        q, k = rng.standard_normal((16, dim)), rng.standard_normal((n, dim))
        v = np.repeat(rng.standard_normal((n // 2, dim)), 2, axis=0) * np.where(np.arange(n) % 2, -1, 1)[:, None]
        s = SCALE * q @ k.T
        e = np.exp(s - s.max(1, keepdims=True)).astype(np.float32).astype(np.float64)
        den = e.sum(1, keepdims=True)
        want, a = e @ v / den, e @ np.abs(v) / den
        hi = _bf16(e)
        rest = _bf16(e - hi)
        off = [np.abs(_bf16((w @ v / den).astype(np.float32)) - want) - bound(want, a) for w in (hi + rest, hi, hi - rest)]
        assert (off[0] <= 0).all()
        assert (off[1] > 0).mean() > 0.3 and (off[2] > 0).mean() > 0.3, (n, [(o > 0).mean() for o in off])


# one row tile and two of every width, dims between them; up to 64 rows of a K/V head (32 of more than 128 dims)
@pytest.mark.gpu
@pytest.mark.parametrize("t,heads,kv,dim", [(1, 4, 1, 64), (3, 16, 2, 64), (1, 64, 1, 64), (1, 8, 2, 128), (1, 40, 1, 128),
                                            (1, 64, 1, 128), (2, 8, 1, 256), (1, 32, 1, 256), (1, 3, 1, 512), (1, 64, 1, 512),
                                            (40, 2, 1, 512), (1, 6, 2, 32), (2, 16, 1, 96), (1, 24, 1, 160), (1, 5, 1, 384)])
@pytest.mark.parametrize("sink", [False, True])
def test_small_outputs_of_large_values(dev, t, heads, kv, dim, sink) -> None:
    from saint_kv import fp4_attention, ops

    lens = [80, 41, 2, 66]
    pool, bt, lens_t = make(dev, lens, 16, kv, dim, seed=dim)
    g = torch.Generator(device=dev).manual_seed(heads)
    k, v = (torch.randn(4, 80, kv, dim, generator=g, device=dev) for _ in range(2))
    v[:, 1::2] = -v[:, 0::2]
    ops.fp4_quant_append(pool, bt, lens_t, k, v, lens_t)
    q = torch.randn(4, t, heads, dim, generator=g, device=dev).to(torch.bfloat16)
    kw = dict(scale=SCALE, sink=torch.randn(heads, generator=g, device=dev) if sink else None)
    on_host = {n: x.cpu().numpy() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    qn, pn, btn, ln = q.cpu().double().numpy(), pool.cpu().numpy(), bt.cpu().numpy(), lens_t.cpu().numpy()
    want = ora.attention(qn, pn, btn, ln, **on_host)
    p = ora.Pages(pn)
    half = p.block * p.dim // 2
    p.flat[:, :, half:2 * half] &= 0x77
    a = ora.attention(qn, pn, btn, ln, **on_host)
    for splits in (0, 1, 3):  # uncut; a workgroup for each; joined pieces
        got = fp4_attention(q, pool, bt, lens_t, splits=splits, **kw).double().cpu().numpy()
        off = np.abs(got - want) - bound(want, a)
        assert (off <= 0).all(), (splits, off.max(), (off > 0).mean())


# views whose rows stay few, and those of 512 dims of any number of rows: 33 of 17 sequences and 200 of four in tiles that waves share
@pytest.mark.gpu
@pytest.mark.parametrize("lens,t,heads,kv,dim", [([80, 41, 2, 66], 1, 64, 1, 64), ([80, 41, 2, 66], 4, 32, 2, 128), ([80, 41, 2, 66], 1, 32, 1, 256),
                                                 ([80, 41, 2, 66], 2, 20, 1, 384), ([80, 41, 2, 66], 1, 64, 1, 512),
                                                 ([80, 41, 5, 66] * 4 + [80], 3, 11, 1, 512), ([80, 41, 33, 66] * 4 + [70], 2, 48, 2, 512),
                                                 ([160, 100, 133, 101], 100, 2, 1, 512)])
@pytest.mark.parametrize("window,first", [(None, 0), (50, 3)])
def test_small_outputs_of_large_values_with_a_view(dev, lens, t, heads, kv, dim, window, first) -> None:
    """As above; a chain given as a tree, and without a tree the window behind first tokens."""
    from saint_kv import fp4_attention, ops

    batch, longest = len(lens), max(lens)
    pool, bt, lens_t = make(dev, lens, 16, kv, dim, seed=dim)
    g = torch.Generator(device=dev).manual_seed(heads)
    k, v = (torch.randn(batch, longest, kv, dim, generator=g, device=dev) for _ in range(2))
    v[:, 1::2] = -v[:, 0::2]
    ops.fp4_quant_append(pool, bt, lens_t, k, v, lens_t)
    q = torch.randn(batch, t, heads, dim, generator=g, device=dev).to(torch.bfloat16)
    chain = np.broadcast_to(np.tri(t, dtype=bool), (batch, t, t))
    tree = torch.as_tensor(ora.pack_masks(chain), device=dev)
    kw = dict(scale=SCALE, window=window, first=first)
    qn, pn, btn, ln = q.cpu().double().numpy(), pool.cpu().numpy(), bt.cpu().numpy(), lens_t.cpu().numpy()
    want = [ora.view_attention(qn, pn, btn, ln, seen=seen, **kw) for seen in (chain, None)]
    p = ora.Pages(pn)
    half = p.block * p.dim // 2
    p.flat[:, :, half:2 * half] &= 0x77
    a = [ora.view_attention(qn, pn, btn, ln, seen=seen, **kw) for seen in (chain, None)]
    for splits in (0, 1, 3):
        for i, masks in enumerate((tree, None)):
            got = fp4_attention(q, pool, bt, lens_t, splits=splits, tree=masks, **kw).double().cpu().numpy()
            off = np.abs(got - want[i]) - bound(want[i], a[i])
            assert (off <= 0).all(), (splits, i, off.max(), (off > 0).mean())
