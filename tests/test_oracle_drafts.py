"""The oracles of drafted tokens and of token probabilities by hand, and the refusals that precede any device work (no GPU;
the pointers are placeholders that a refused call never reads)."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from oracle import drafts
from oracle import fp4_cache as ora
from oracle.token_logprobs import token_logprobs

FAKE = 4096  # aligned, never dereferenced


def test_accepts_along_the_picks() -> None:
    # 0 -> 1 (token 7), 0 -> 2 (token 8), 2 -> 3 (token 9), 2 -> 4 (token 9), 4 -> 5
    parents = np.array([[-1, 0, 0, 2, 2, 4]] * 4)
    tokens = np.array([[5, 7, 8, 9, 9, 1]] * 4)
    picks = np.array([[8, 0, 9, 1, 1, 3], [6, 0, 9, 1, 1, 3], [8, 0, 9, 1, 1, 3], [7, 0, 9, 1, 1, 3]])
    path, n_keep, following = drafts.accept(parents, tokens, picks, np.array([6, 6, 3, 0]))
    assert path.tolist() == [[0, 2, 3, -1, -1, -1], [0] + [-1] * 5, [0, 2] + [-1] * 4, [-1] * 6]
    assert n_keep.tolist() == [3, 1, 2, 0] and following.tolist() == [1, 6, 9, -1]


def _cache():
    """Two sequences of 35 and 20 tokens in pages of 16, byte i of a row telling its position."""
    pool = np.zeros((8, 16, 2, 34), dtype=np.uint8)
    bt = np.array([[3, 1, 6], [0, 4, -1]], dtype=np.int32)
    lens = np.array([35, 20], dtype=np.int32)
    p = ora.Pages(pool)
    for b in range(2):
        for pos in range(lens[b]):
            for kv in range(2):
                for where in p._at(pos % 16, kv):
                    p.flat[bt[b, pos // 16], :, where] = 100 * b + pos
    stack = np.array([2, 5, 7, 0, 0, 0, 0, 0], dtype=np.int32)
    return pool, bt, lens, stack


def _positions(pool, bt, lens, b):
    p = ora.Pages(pool)
    return [int(p.flat[bt[b, i // 16], 1, p._at(i % 16, 1)[1]][0]) for i in range(lens[b])]


def test_kept_tokens_move_together() -> None:
    pool, bt, lens, stack = _cache()
    path = np.array([[0, 2, 3], [1, -1, -1]])
    top, status = drafts.keep(stack, 3, bt, lens, np.array([5, 3]), path, np.array([3, 1]), [pool])
    assert (top, status) == (3, 0) and lens.tolist() == [33, 18]
    assert _positions(pool, bt, lens, 0) == [*range(30), 30, 32, 33]
    assert _positions(pool, bt, lens, 1) == [*range(100, 117), 118]


def test_pages_behind_return_last_first() -> None:
    pool, bt, lens, stack = _cache()
    path = np.full((2, 40), -1)
    top, status = drafts.keep(stack, 3, bt, lens, np.array([34, 20]), path, np.array([0, 0]), [pool])
    assert (top, status) == (7, 0) and lens.tolist() == [1, 0]
    assert stack[:7].tolist() == [2, 5, 7, 6, 1, 4, 0] and bt.tolist() == [[3, -1, -1], [-1, -1, -1]]


@pytest.mark.parametrize("n_new,path,n_keep,refs,status", [
    ([5, 3], [[2, 0], [0, 1]], [2, 2], None, 4), ([5, 3], [[0, 5], [0, 1]], [2, 2], None, 4),
    ([5, 3], [[0, 1], [0, 1]], [2, 3], None, 4), ([36, 3], [[0, 1], [0, 1]], [2, 2], None, 4),
    ([5, 3], [[1, 2], [0, 1]], [2, 2], 1, 4), ([5, 3], [[0, 1], [0, 1]], [2, 2], 6, 4),
    ([5, 3], [[0, 1], [1, 2]], [2, 2], 3, 0)])
def test_refused_keeps_write_nothing(n_new, path, n_keep, refs, status) -> None:
    pool, bt, lens, stack = _cache()
    before = [x.copy() for x in (pool, bt, lens, stack)]
    r = np.zeros(8, dtype=np.int32)
    if refs is not None:
        r[refs] = 1
    got = drafts.keep(stack, 3, bt, lens, np.array(n_new), np.array(path), np.array(n_keep), [pool], r)
    assert got[1] == status
    if status:
        assert all(np.array_equal(x, y) for x, y in zip((pool, bt, lens, stack), before))


def test_probabilities_by_hand() -> None:
    ninf, nan = -math.inf, math.nan
    x = np.array([[0.0, math.log(2.0), ninf, 0.0], [1.0, 1.0, 1.0, 1.0], [ninf] * 4, [0.0, nan, 5.0, nan], [-0.0, 0.0, ninf, 3e38]])
    lp, h, ids, best = token_logprobs(x, np.array([1, -1, 0, 2, 4]), 3)
    assert np.allclose(lp[:2], [math.log(0.5), 0.0]) and np.isnan(lp[2:]).all()
    assert np.allclose(h[:2], [1.5 * math.log(2.0), math.log(4.0)]) and np.isnan(h[2:4]).all() and h[4] == 0
    assert ids.tolist() == [[1, 0, 3], [0, 1, 2], [0, 1, 2], [1, 3, 2], [3, 0, 1]]
    assert np.allclose(best[0], np.log([0.5, 0.25, 0.25])) and best[4, 0] == 0


def _refused(rc: int, text: str) -> None:
    from saint_kv import _lib

    assert rc == _lib.SKV_EINVAL and text in _lib.last_error(), (rc, _lib.last_error())


def test_bad_trees_are_refused() -> None:
    from saint_kv import _lib

    lib = _lib.load()
    ids = _lib.TokenIds(FAKE, 4, 1, 0, 0)
    for batch, nodes, text in ((-1, 4, "batch"), (65536, 4, "batch"), (2, 0, "n_nodes"), (2, 1025, "n_nodes")):
        _refused(lib.skv_draft_tree(FAKE, None, batch, nodes, FAKE, FAKE, None), text)
        _refused(lib.skv_accept_drafts(FAKE, ctypes.byref(ids), ctypes.byref(ids), None, batch, nodes, FAKE, FAKE, FAKE, None), text)
    for missing in (0, 4, 5):
        args = [FAKE, None, 2, 4, FAKE, FAKE, None]
        args[missing] = None
        _refused(lib.skv_draft_tree(*args), "NULL")
    none = _lib.TokenIds(None, 4, 1, 0, 0)
    _refused(lib.skv_accept_drafts(FAKE, ctypes.byref(none), ctypes.byref(ids), None, 2, 4, FAKE, FAKE, FAKE, None), "NULL")
    _refused(lib.skv_accept_drafts(FAKE, None, ctypes.byref(ids), None, 2, 4, FAKE, FAKE, FAKE, None), "NULL")
    assert lib.skv_draft_tree(None, None, 0, 4, None, None, None) == 0
    assert lib.skv_accept_drafts(None, ctypes.byref(none), ctypes.byref(none), None, 0, 4, None, None, None, None) == 0


def test_bad_keeps_are_refused() -> None:
    from saint_kv import _lib

    lib = _lib.load()

    def keep(cache=None, pools=1, stride=4, n_uni=4, ws=1 << 20, **over):
        c = _lib.Fp4Cache(**{**dict(pool=None, block_size=16, n_pages=8, n_kv_heads=2, head_dim=128, block_table=None,
                                    bt_stride=4, batch=3), **(cache or {})})
        arr = (ctypes.c_void_p * 40)(*[FAKE] * 40)
        if "pool" in over:
            arr[0] = over["pool"]
        p = {k: over.get(k, FAKE) for k in ("stack", "top", "bt", "lens", "path", "n_keep", "status", "wsp")}
        return lib.skv_keep_tokens(p["stack"], p["top"], None, ctypes.byref(c), p["bt"], p["lens"], None, n_uni, p["path"],
                                   stride, p["n_keep"], ctypes.cast(arr, ctypes.c_void_p), pools, p["status"], p["wsp"], ws, None)

    for over, text in ((dict(cache=dict(batch=4097)), "batch"), (dict(cache=dict(block_size=8)), "block_size"),
                       (dict(cache=dict(head_dim=40)), "head_dim"), (dict(cache=dict(n_pages=0)), "geometry"),
                       (dict(pools=0), "n_pools"), (dict(pools=33), "n_pools"), (dict(stride=0), "path_stride"),
                       (dict(stride=1025), "path_stride"), (dict(n_uni=-1), "n_new"), (dict(ws=3 * 4 * 16 - 1), "workspace"),
                       (dict(wsp=FAKE + 8), "workspace"), (dict(wsp=None), "workspace"), (dict(pool=None), "NULL"),
                       (dict(pool=FAKE + 8), "aligned")):
        _refused(keep(**over), text)
    for name in ("stack", "top", "lens", "path", "n_keep", "status", "bt"):
        _refused(keep(**{name: None}), "NULL")
    assert keep(cache=dict(batch=0)) == 0
    assert lib.skv_keep_tokens_workspace(3, 7) == 3 * 7 * 16 and lib.skv_keep_tokens_workspace(4097, 7) == -1


def test_bad_logits_are_refused() -> None:
    from saint_kv import _lib

    lib = _lib.load()
    ids = _lib.TokenIds(FAKE, 0, 1, 1, 0)

    def call(rows=4, vocab=100, stride=100, fmt=0, top=5, logits=FAKE, tokens=ids, lp=FAKE, h=FAKE, ti=FAKE, tl=FAKE, ws=None, n=0):
        return lib.skv_token_logprobs(logits, rows, vocab, stride, fmt, None if tokens is None else ctypes.byref(tokens), top, lp, h,
                                      ti, tl, ws, n, None)

    for over, text in ((dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"), (dict(vocab=0), "vocab"),
                       (dict(vocab=(1 << 24) + 1), "vocab"), (dict(fmt=3), "format"), (dict(fmt=-1), "format"), (dict(top=-1), "top"),
                       (dict(top=65), "top"), (dict(top=101), "top"), (dict(vocab=4, top=5), "top"), (dict(logits=None), "NULL"),
                       (dict(h=None), "NULL"), (dict(lp=None), "NULL"), (dict(ti=None), "NULL"), (dict(tl=None), "NULL"),
                       (dict(logits=FAKE + 1), "aligned"), (dict(logits=FAKE + 2, fmt=2), "aligned"), (dict(stride=-1), "row_stride"),
                       (dict(tokens=_lib.TokenIds(None, 0, 1, 0, 0)), "NULL"), (dict(rows=1, vocab=1 << 22), "workspace"),
                       (dict(rows=1, vocab=1 << 22, ws=FAKE, n=8), "workspace"),
                       (dict(rows=1, vocab=1 << 22, ws=FAKE + 8, n=1 << 20), "workspace")):
        _refused(call(**over), text)
    assert call(rows=0) == 0
    assert lib.skv_token_logprobs_workspace(1 << 16, 100, 0, 5) == 0  # rows enough for the device
    assert lib.skv_token_logprobs_workspace(1, 1 << 20, 0, 5) > 0 and lib.skv_token_logprobs_workspace(1, 0, 0, 5) == -1


def test_sizes_past_a_launch_are_refused() -> None:
    """2^32 work-items, and a table whose pages a 32-bit count could not number."""
    from saint_kv import _lib

    lib = _lib.load()
    ids = _lib.TokenIds(FAKE, 0, 1, 1, 0)
    most = (1 << 24) - 1  # rows of a workgroup of 256 each
    assert lib.skv_token_logprobs_workspace(most, 8, 0, 2) == 0 and lib.skv_token_logprobs_workspace(most + 1, 8, 0, 2) == -1
    _refused(lib.skv_token_logprobs(FAKE, most + 1, 8, 8, 0, ctypes.byref(ids), 2, FAKE, FAKE, FAKE, FAKE, None, 0, None),
             "too many rows")
    c = _lib.Fp4Cache(pool=None, block_size=16, n_pages=8, n_kv_heads=2, head_dim=128, block_table=None, bt_stride=1 << 20,
                      batch=2048)
    pools = (ctypes.c_void_p * 1)(FAKE)
    rc = lib.skv_keep_tokens(FAKE, FAKE, None, ctypes.byref(c), FAKE, FAKE, None, 4, FAKE, 4, FAKE,
                             ctypes.cast(pools, ctypes.c_void_p), 1, FAKE, FAKE, 1 << 20, None)
    _refused(rc, "block_table")
