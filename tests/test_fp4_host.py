"""Argument checks of the 4-bit cache and of forks that precede any device work (no GPU):
the pointers are placeholders that a refused call never reads."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

FAKE = 4096  # aligned, never dereferenced


def _cache(**over):
    from saint_kv import _lib

    c = dict(pool=FAKE, block_size=16, n_pages=8, n_kv_heads=2, head_dim=128, block_table=FAKE, bt_stride=4, batch=3)
    c.update(over)
    return _lib.Fp4Cache(**c)


def _rows(**over):
    from saint_kv import _lib

    return _lib.Fp4Rows(**{**dict(data=FAKE, seq_stride=4096, tok_stride=512, head_stride=256), **over})


def _refused(rc: int, text: str) -> None:
    from saint_kv import _lib

    assert rc == _lib.SKV_EINVAL and text in _lib.last_error(), (rc, _lib.last_error())


BAD_CACHES = [(dict(block_size=8), "block_size"), (dict(block_size=24), "block_size"), (dict(block_size=0), "block_size"),
              (dict(n_kv_heads=0), "n_kv_heads"), (dict(n_kv_heads=257), "n_kv_heads"), (dict(head_dim=48), "head_dim"),
              (dict(head_dim=544), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(batch=-1), "batch"),
              (dict(batch=70000), "batch"), (dict(n_pages=0), "geometry"), (dict(bt_stride=0), "geometry"),
              (dict(bt_stride=(1 << 20) + 1), "geometry"), (dict(pool=None), "NULL"), (dict(pool=FAKE + 8), "aligned"),
              (dict(block_table=None), "NULL")]


@pytest.mark.parametrize("over,text", BAD_CACHES)
def test_a_bad_cache_is_refused_everywhere(over: dict, text: str) -> None:
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    c = _cache(**over)
    _refused(lib.skv_fp4_quant_append(ctypes.byref(c), FAKE, None, 1, ctypes.byref(_rows()), ctypes.byref(_rows()), 4, 0,
                                      None), text)
    _refused(lib.skv_fp4_gather(ctypes.byref(c), FAKE, None, 1, ctypes.byref(_rows()), ctypes.byref(_rows()), 4, None),
             text)
    d = Fp4AttentionDesc(cache=c, seq_lens=FAKE, n_queries=1, n_heads=4, q=FAKE, out=FAKE)
    _refused(lib.skv_fp4_attention(ctypes.byref(d), None, 0, None), text)


def test_page_bytes() -> None:
    from saint_kv import _lib

    lib = _lib.load()
    assert lib.skv_fp4_page_bytes(16, 1, 32) == 16 * 34
    assert lib.skv_fp4_page_bytes(64, 8, 128) == 64 * 8 * 136
    assert lib.skv_fp4_page_bytes(8, 1, 32) == -1 and lib.skv_fp4_page_bytes(16, 1, 33) == -1


@pytest.mark.parametrize("over", [dict(data=FAKE + 4), dict(seq_stride=8), dict(tok_stride=24), dict(head_stride=2),
                                  dict(data=None)])
def test_bad_rows_are_refused(over: dict) -> None:
    from saint_kv import _lib

    lib = _lib.load()
    c = _cache()
    for k, v in ((_rows(**over), _rows()), (_rows(), _rows(**over))):
        text = "NULL" if "data" in over and over["data"] is None else "aligned"
        _refused(lib.skv_fp4_quant_append(ctypes.byref(c), FAKE, None, 1, ctypes.byref(k), ctypes.byref(v), 4, 0, None), text)
        _refused(lib.skv_fp4_gather(ctypes.byref(c), FAKE, None, 1, ctypes.byref(k), ctypes.byref(v), 4, None), text)


def test_bad_counts_are_refused() -> None:
    from saint_kv import _lib

    lib = _lib.load()
    c, k = _cache(), _rows()
    _refused(lib.skv_fp4_quant_append(ctypes.byref(c), FAKE, None, -1, ctypes.byref(k), ctypes.byref(k), 4, 0, None), "n_new")
    _refused(lib.skv_fp4_gather(ctypes.byref(c), None, None, 1, ctypes.byref(k), ctypes.byref(k), 4, None), "NULL")
    _refused(lib.skv_fp4_gather(ctypes.byref(c), FAKE, None, 1, ctypes.byref(k), ctypes.byref(k), -1, None), "rows")


@pytest.mark.parametrize("over,text", [
    (dict(n_heads=0), "n_heads"), (dict(n_heads=5), "n_heads"), (dict(n_heads=1026), "n_heads"),
    (dict(n_queries=0), "n_queries"), (dict(n_queries=70000), "n_queries"), (dict(window=-1), "window"),
    (dict(window=(1 << 24) + 1), "window"), (dict(max_len=-1), "max_len"), (dict(splits=-1), "splits"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(softcap=float("inf")), "softcap"),
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(seq_lens=None), "NULL"), (dict(q=FAKE + 2), "aligned"),
    (dict(out=FAKE + 8), "aligned"), (dict(q_head_stride=100), "aligned"),
])
def test_a_bad_attention_is_refused(over: dict, text: str) -> None:
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    assert lib.skv_fp4_attention_desc_size() == ctypes.sizeof(Fp4AttentionDesc)
    args = dict(cache=_cache(), seq_lens=FAKE, n_queries=1, n_heads=4, q=FAKE, out=FAKE)
    args.update(over)
    d = Fp4AttentionDesc(**args)
    _refused(lib.skv_fp4_attention(ctypes.byref(d), FAKE, 1 << 40, None), text)


def test_an_empty_batch_is_nothing_to_do() -> None:
    from saint_kv import _lib
    from saint_kv.fp4 import Fp4AttentionDesc

    lib = _lib.load()
    c = _cache(batch=0, pool=None, block_table=None)
    k = _rows(data=None)
    assert lib.skv_fp4_quant_append(ctypes.byref(c), FAKE, None, 1, ctypes.byref(k), ctypes.byref(k), 4, 0, None) == 0
    d = Fp4AttentionDesc(cache=c, n_queries=1, n_heads=4)
    assert lib.skv_fp4_attention(ctypes.byref(d), None, 0, None) == 0


def test_bad_forks_are_refused() -> None:
    from saint_kv import _lib

    lib = _lib.load()
    pool = (_lib.PoolRef * 1)(_lib.PoolRef(FAKE, 1024))

    def fork(n_pages=8, refs=FAKE, bt_stride=4, batch=3, block=16, n=2, pools=pool, n_pools=1, status=FAKE):
        return lib.skv_fork(FAKE, FAKE, n_pages, refs, FAKE, bt_stride, FAKE, batch, block, FAKE, FAKE, n,
                            ctypes.cast(pools, ctypes.c_void_p), n_pools, status, None)

    for over, text in ((dict(n=4097), "n_forks"), (dict(n=-1), "n_forks"), (dict(batch=5000), "batch"),
                       (dict(batch=0), "empty batch"), (dict(block=0), "block_size"), (dict(bt_stride=0), "bt_stride"),
                       (dict(n_pages=0), "n_pages"), (dict(n_pools=33), "n_pools"), (dict(refs=None), "NULL"),
                       (dict(status=None), "NULL"), (dict(pools=(_lib.PoolRef * 1)(_lib.PoolRef(FAKE, 8))), "aligned")):
        _refused(fork(**over), text)
    assert fork(n=0) == 0
    arr = ctypes.cast(pool, ctypes.c_void_p)
    _refused(lib.skv_copy_slots(arr, 1, 4, None, FAKE, 2, None), "NULL")
    _refused(lib.skv_copy_slots(arr, 1, 4, FAKE, FAKE, 70000, None), "n_forks")
    _refused(lib.skv_copy_slots(ctypes.cast((_lib.PoolRef * 1)(_lib.PoolRef(FAKE, 0)), ctypes.c_void_p), 1, 4, FAKE, FAKE, 2,
                                None), "slot size")
    assert lib.skv_copy_slots(arr, 1, 4, FAKE, FAKE, 0, None) == 0


def test_bad_shared_releases_and_compactions_are_refused() -> None:
    from saint_kv import _lib

    lib = _lib.load()

    def release(refs=FAKE, mask=FAKE, batch=3, block=16, stride=4, pages=8):
        return lib.skv_release_shared(FAKE, FAKE, pages, refs, FAKE, stride, FAKE, mask, batch, block, FAKE, None)

    for over, text in ((dict(refs=None), "NULL"), (dict(mask=None), "NULL"), (dict(batch=5000), "batch"),
                       (dict(block=0), "block_size"), (dict(stride=1 << 31), "bt_stride"), (dict(pages=0), "n_pages")):
        _refused(release(**over), text)
    assert release(batch=0) == 0
    pool = ctypes.cast((_lib.PoolRef * 1)(_lib.PoolRef(FAKE, 1024)), ctypes.c_void_p)
    _refused(lib.skv_compact_shared(pool, 1, FAKE, 4, FAKE, 3, 16, 8, FAKE, FAKE, None, FAKE, FAKE, None), "refs")
    _refused(lib.skv_compact_shared(pool, 0, FAKE, 4, FAKE, 3, 16, 8, FAKE, FAKE, FAKE, FAKE, FAKE, None), "n_pools")


def test_check_forks() -> None:
    from saint_kv.fp4 import check_forks

    lens = np.array([5, 0, 0, 7])
    src, dst = check_forks([0, 0], [1, 2], lens)
    assert src.tolist() == [0, 0] and dst.tolist() == [1, 2]
    assert check_forks(3, 1, lens)[0].tolist() == [3]
    for s, d, error in (([0, 0], [1], ValueError), ([0], [4], ValueError), ([-1], [1], ValueError),
                        ([0, 3], [1, 1], ValueError), ([0], [3], RuntimeError), ([0], [0], RuntimeError)):
        with pytest.raises(error):
            check_forks(s, d, lens)


def test_the_caches_refuse_a_cpu_and_bad_sizes() -> None:
    import torch

    from saint_kv import Fp4TokenCache, fp4_attention, ops

    with pytest.raises(RuntimeError, match="GPU"):
        Fp4TokenCache(1, 1, 16, 1, 64, device="cpu")
    for bad in (dict(layers=0), dict(layers=17), dict(batch=0), dict(batch=5000), dict(max_len=0)):
        with pytest.raises(ValueError):
            Fp4TokenCache(**{**dict(layers=1, batch=1, max_len=16, n_kv_heads=1, head_dim=64, device="cpu"), **bad})
    t = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CPU"):
        fp4_attention(t, t, t, t)
    with pytest.raises(RuntimeError, match="CPU"):
        ops.fp4_cache(t, t)
    for bs, heads, dim in ((8, 1, 64), (16, 0, 64), (16, 1, 40)):
        with pytest.raises(ValueError):
            ops.fp4_pool(2, bs, heads, dim, "cpu")
