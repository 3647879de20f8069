"""Arguments of the 4-bit cache and of forks at the ends of what they may be, refused or sorted out on
the host (no GPU; the pointers are placeholders that a refused call never reads)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

FAKE = 4096  # aligned, never dereferenced


@pytest.mark.parametrize("batch,kv_heads", [(1, 1), (3, 2), (8, 2), (4, 1), (512, 16)])
@pytest.mark.parametrize("splits", [1 << 24, (1 << 24) + 1, 1 << 32, 1 << 58, 1 << 59, 1 << 60, 1 << 62, (1 << 63) - 1])
def test_splits_past_any_launch_are_refused(batch: int, kv_heads: int, splits: int) -> None:
    """Their product with the batch's items wraps to a small, zero or negative number of workgroups."""
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    cache = _lib.Fp4Cache(FAKE, 64, 4096, kv_heads, 128, FAKE, 2048, batch)
    d = Fp4AttentionDesc(cache=cache, seq_lens=FAKE, n_queries=1, n_heads=kv_heads, q=FAKE, out=FAKE, splits=splits)
    assert lib.skv_fp4_attention_workspace(ctypes.byref(d)) == -1
    assert "splits" in _lib.last_error()
    assert lib.skv_fp4_attention(ctypes.byref(d), FAKE, (1 << 63) - 1, None) == _lib.SKV_EINVAL
    assert "splits" in _lib.last_error()


def test_the_most_splits() -> None:
    """Up to the bound the workspace holds two pieces of every run: [rows] of m, l and 128 dims, in fp32."""
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    for batch, kv_heads, splits in ((1, 1, (1 << 24) - 1), (4, 2, (1 << 21) - 1), (8, 2, 3)):
        cache = _lib.Fp4Cache(FAKE, 64, 4096, kv_heads, 128, FAKE, 2048, batch)
        d = Fp4AttentionDesc(cache=cache, seq_lens=FAKE, n_queries=1, n_heads=kv_heads, q=FAKE, out=FAKE, splits=splits)
        sched = -(-(batch + 2) * 4 // 16) * 16
        assert lib.skv_fp4_attention_workspace(ctypes.byref(d)) == sched + 2 * splits * batch * kv_heads * 16 * 132 * 4


def test_no_forks_need_no_indices() -> None:
    """An empty device array has no address."""
    from saint_kv import _lib

    lib = _lib.load()

    def fork(n, src, dst):
        return lib.skv_fork(FAKE, FAKE, 8, FAKE, FAKE, 4, FAKE, 3, 16, src, dst, n, None, 0, FAKE, None)

    assert fork(0, None, None) == 0
    for src, dst in ((None, FAKE), (FAKE, None)):
        assert fork(1, src, dst) == _lib.SKV_EINVAL and "NULL" in _lib.last_error()


def test_forks_of_empty_sequences_are_left_out() -> None:
    """Also where the empty source is another fork's destination: all copies are of what was there before."""
    from saint_kv.fp4 import check_forks

    src, dst = check_forks([0, 1, 2, 3], [1, 4, 5, 2], np.array([5, 0, 0, 7, 0, 0]))
    assert src.tolist() == [0, 3] and dst.tolist() == [1, 2]


def test_a_cache_that_its_calls_would_refuse() -> None:
    """Sizes that only a later append, release or compaction would refuse."""
    from saint_kv import Fp4TokenCache

    ok = dict(layers=1, batch=2, max_len=4096, n_kv_heads=1, head_dim=64, device="cpu")
    for bad, text in ((dict(max_len=(1 << 24) + 1), "tokens"), (dict(max_len=(1 << 24) - 8, block_size=96), "tokens"),
                      (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 24), "n_pages"), (dict(n_pages=-4), "n_pages"),
                      (dict(batch=4096, max_len=1 << 18, block_size=16), "n_pages"),
                      (dict(batch=4096, max_len=1 << 23, block_size=16, n_pages=1000), "table")):
        with pytest.raises(ValueError, match=text):
            Fp4TokenCache(**{**ok, **bad})
    for good in (dict(max_len=1 << 24), dict(n_pages=(1 << 24) - 1), dict(batch=4096, max_len=1 << 20, n_pages=1000)):
        with pytest.raises(RuntimeError, match="GPU"):  # what is left to refuse is the device
            Fp4TokenCache(**{**ok, **good})


def test_slots_past_a_launch_are_refused() -> None:
    from saint_kv import _lib

    lib = _lib.load()
    arr = (_lib.PoolRef * 1)(_lib.PoolRef(FAKE, (1 << 37) + 16))
    assert lib.skv_copy_slots(ctypes.cast(arr, ctypes.c_void_p), 1, 4, FAKE, FAKE, 2, None) == _lib.SKV_EINVAL
    assert "slot size" in _lib.last_error()


@pytest.mark.parametrize("page_bytes,bt_stride,text", [(1 << 38, 4, "pages too large"), ((1 << 38) - (1 << 14), 4, "pages and"),
                                                       ((1 << 38) - (1 << 34), (1 << 31) - 1, "pages and")])
def test_forks_past_a_launch_are_refused(page_bytes: int, bt_stride: int, text: str) -> None:
    """Before their pages are popped: a copy launch that then fails would leave them lost."""
    from saint_kv import _lib

    lib = _lib.load()
    pool = ctypes.cast((_lib.PoolRef * 1)(_lib.PoolRef(FAKE, page_bytes)), ctypes.c_void_p)
    rc = lib.skv_fork(FAKE, FAKE, 8, FAKE, FAKE, bt_stride, FAKE, 3, 16, FAKE, FAKE, 2, pool, 1, FAKE, None)
    assert rc == _lib.SKV_EINVAL and text in _lib.last_error()
