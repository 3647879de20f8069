"""Softcapped attention over the 4-bit pages for caps of every size: a cap far above the scores
leaves them as they are, one far below holds them all at its ends.

The bound is that of test_gpu_fp4_attention.py, whose share for the scores' own error (a quarter of
2^-8 of A) takes a relative error of a score |s| <= 60 of up to 2^-10 / 60 = 2^-16.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_fp4_attention import check, make

pytestmark = pytest.mark.gpu


# one row tile, several, shared tiles; every padded width, dims between them among them
@pytest.mark.parametrize("t,heads,kv,dim", [(1, 4, 2, 128), (1, 40, 1, 64), (40, 8, 2, 64), (70, 2, 1, 256), (2, 3, 1, 512),
                                            (3, 4, 2, 96)])
@pytest.mark.parametrize("cap", [1e-3, 2.0, 30.0, 1e3, 1e4, 1e5, 1e6, 1e8, 1e15, 1e22, 1e30])
def test_caps_of_every_size(dev, t, heads, kv, dim, cap) -> None:
    from saint_kv import fp4_attention

    lens = [200, 77]
    pool, bt, lens_t = make(dev, lens, 16, kv, dim, seed=t)
    g = torch.Generator(device=dev).manual_seed(dim)
    q = (4 * torch.randn(2, t, heads, dim, generator=g, device=dev)).to(torch.bfloat16)  # scores of up to about 20
    sink = torch.randn(heads, generator=g, device=dev)
    for kw in (dict(softcap=cap), dict(softcap=cap, sink=sink, window=50), dict(softcap=cap, scale=1e-3)):
        check(fp4_attention(q, pool, bt, lens_t, **kw), q, pool, bt, lens_t, **kw)


@pytest.mark.parametrize("t,heads", [(1, 4), (1, 40), (40, 8)])
def test_scores_on_both_sides_of_the_cap(dev, t, heads) -> None:
    """Scores from far below a cap to far above it in one row, and ones that fp32 cannot hold."""
    from saint_kv import fp4_attention

    pool, bt, lens = make(dev, [300], 16, 1, 64)
    q = torch.randn(1, t, heads, 64, generator=torch.Generator(device=dev).manual_seed(3), device=dev)
    q *= torch.logspace(-3, 2, heads, device=dev)[:, None]
    q = q.to(torch.bfloat16)
    for cap in (0.5, 8.0, 60.0):
        check(fp4_attention(q, pool, bt, lens, softcap=cap), q, pool, bt, lens, softcap=cap)
    q[:] = 3e38  # products past fp32 become infinities, the cap's ends
    got = fp4_attention(q, pool, bt, lens, softcap=5.0)
    assert torch.isfinite(got).all()
