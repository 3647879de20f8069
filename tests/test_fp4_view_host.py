"""Views of the 4-bit cache: the oracle's masks and histories by hand, and the refusals that precede any device work (no
GPU; the pointers are placeholders that a refused call never reads)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import fp4_cache as ora

FAKE = 4096  # aligned, never dereferenced


def test_masks_of_a_small_tree() -> None:
    # 0 - 1 - 3, 1 - 4, 0 - 2; 5 a second root; 6 below a later node, 7 below it
    parents = np.array([[-1, 0, 0, 1, 1, -1, 7, 6]])
    seen = ora.tree_masks(parents, np.array([8]))[0]
    want = {0: [0], 1: [0, 1], 2: [0, 2], 3: [0, 1, 3], 4: [0, 1, 4], 5: [5], 6: [], 7: []}
    for t, up in want.items():
        assert np.flatnonzero(seen[t]).tolist() == up
    assert ora.pack_masks(seen[None])[0, :, 0].tolist() == [1, 3, 5, 11, 19, 32, 0, 0]
    assert not ora.tree_masks(parents, np.array([2]))[0, 2:].any()


def test_masks_past_a_word() -> None:
    parents = np.arange(-1, 69)[None]
    words = ora.pack_masks(ora.tree_masks(parents, np.array([70])))
    assert words.shape == (1, 70, 2)
    assert words[0, 63].tolist() == [-1, 0] and words[0, 65].tolist() == [-1, 3]


def test_histories() -> None:
    row = np.array([True, False, True, False])
    assert ora.history(10, 4, 2, row) == [0, 1, 2, 3, 4, 5, 6, 8]
    assert ora.history(10, 4, 2, None) == list(range(9))
    assert ora.history(10, 4, 2, row & False) == []
    assert ora.history(3, 4, 2, row) == [] and ora.history(3, 4, 2, None) == [0, 1]


def test_an_oracle_of_a_view_of_all_is_the_plain_one() -> None:
    rng = np.random.default_rng(0)
    pool = np.zeros((3, 16, 1, 34), dtype=np.uint8)
    bt, lens = np.array([[2, 0], [1, -1]]), np.array([20, 7])
    k, v = rng.standard_normal((2, 2, 20, 1, 32))
    ora.append(pool, bt, lens, k, v, lens)
    q = rng.standard_normal((2, 3, 2, 32))
    chain = np.broadcast_to(np.tri(3, dtype=bool), (2, 3, 3))
    for window in (None, 4):
        want = ora.attention(q, pool, bt, lens, window=window)
        assert np.allclose(ora.view_attention(q, pool, bt, lens, window=window), want)
        assert np.allclose(ora.view_attention(q, pool, bt, lens, window=window, seen=chain), want)
    assert np.allclose(ora.view_attention(q, pool, bt, lens, window=4, first=30), ora.attention(q, pool, bt, lens))


@pytest.mark.parametrize("over,text", [(dict(first=-1), "first"), (dict(first=(1 << 24) + 1), "first"),
                                       (dict(tree=FAKE, tree_words=2), "words"), (dict(tree=FAKE, tree_words=0), "words"),
                                       (dict(tree=FAKE + 4, tree_words=1), "aligned")])
def test_bad_views_are_refused(over: dict, text: str) -> None:
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    cache = _lib.Fp4Cache(FAKE, 64, 4096, 2, 128, FAKE, 2048, 3)
    d = Fp4AttentionDesc(cache=cache, seq_lens=FAKE, n_queries=5, n_heads=4, q=FAKE, out=FAKE)
    v = _lib.Fp4View(**over)
    assert lib.skv_fp4_attention_view_workspace(ctypes.byref(d), ctypes.byref(v)) == -1 and text in _lib.last_error()
    assert lib.skv_fp4_attention_view(ctypes.byref(d), ctypes.byref(v), FAKE, 1 << 40, None) == _lib.SKV_EINVAL
    assert text in _lib.last_error()


def test_large_trees_and_missing_views_are_refused() -> None:
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    cache = _lib.Fp4Cache(FAKE, 64, 4096, 2, 128, FAKE, 2048, 3)
    d = Fp4AttentionDesc(cache=cache, seq_lens=FAKE, n_queries=1025, n_heads=4, q=FAKE, out=FAKE)
    assert lib.skv_fp4_attention_view_workspace(ctypes.byref(d), ctypes.byref(_lib.Fp4View(FAKE, 17, 0))) == -1
    assert "1024" in _lib.last_error()
    assert lib.skv_fp4_attention_view_workspace(ctypes.byref(d), ctypes.byref(_lib.Fp4View(None, 0, 4))) > 0
    assert lib.skv_fp4_attention_view_workspace(ctypes.byref(d), None) == -1 and "NULL" in _lib.last_error()
    assert lib.skv_fp4_attention_view(ctypes.byref(d), None, None, 0, None) == _lib.SKV_EINVAL


@pytest.mark.parametrize("window,first,t,heads", [(128, 4, 1, 16), (300, 0, 9, 4), (64, 100, 99, 4), (1, 1, 1, 1)])
def test_short_views_need_no_workspace(window: int, first: int, t: int, heads: int) -> None:
    """A window, a tree and first tokens of few tiles are not cut."""
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    cache = _lib.Fp4Cache(FAKE, 64, 4096, 1, 128, FAKE, 2048, 3)
    d = Fp4AttentionDesc(cache=cache, seq_lens=FAKE, n_queries=t, n_heads=heads, q=FAKE, out=FAKE, window=window)
    for v in (_lib.Fp4View(FAKE, -(-t // 64), first), _lib.Fp4View(None, 0, first)):
        assert lib.skv_fp4_attention_view_workspace(ctypes.byref(d), ctypes.byref(v)) == 0
