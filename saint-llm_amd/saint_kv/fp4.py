"""A token cache held in 4 bits, and the attention over it.

Keys and values of several K/V heads in pages of e2m1 codes with a power-of-two
scale per 32 dims (``skv_fp4_cache`` in include/saintkv.h): 17/32 of a byte per
value, 3.8 times less than bf16.  ``ops.fp4_quant_append`` writes them,
``ops.fp4_gather`` reads them back, ``fp4_attention`` attends over them in
place, for single tokens and for the tokens of a prompt's chunk alike.
``Fp4TokenCache`` keeps the pages, block table and free list of a stack of
layers, and forks, releases and compacts its sequences.

The reference keeps a layer's raw K/V rows at full width and attends over them
with the window as a mask (kv_cache.py:59-83, swa.py:107-137); its
mixed-precision storage is a plan (``saint_llm_inference/__init__.py:9``).
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch

from saint_kv import _lib, ops
from saint_kv.ops import _launch, _require_gpu, _require_i32, _same_device

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
MAX_LAYERS = 16
MAX_BATCH = 4096
STATUS_WORDS = 64


class Fp4AttentionDesc(ctypes.Structure):
    """Mirror of skv_fp4_attention_desc (include/saintkv.h)."""

    _fields_ = [
        ("cache", _lib.Fp4Cache), ("seq_lens", _P), ("n_new", _P), ("n_queries", _I64), ("n_heads", _I64),
        ("q", _P), ("q_seq_stride", _I64), ("q_tok_stride", _I64), ("q_head_stride", _I64),
        ("out", _P), ("sink", _P), ("window", _I64), ("max_len", _I64), ("splits", _I64),
        ("scale", ctypes.c_float), ("softcap", ctypes.c_float),
    ]


_layout_checked = False


def _check_layout() -> None:
    global _layout_checked
    if not _layout_checked:
        size = _lib.load().skv_fp4_attention_desc_size()
        if size != ctypes.sizeof(Fp4AttentionDesc):
            raise RuntimeError(f"skv_fp4_attention_desc layout mismatch: library {size} vs ctypes "
                               f"{ctypes.sizeof(Fp4AttentionDesc)}")
        _layout_checked = True


def fp4_attention(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                  n_new: torch.Tensor | None = None, window: int | None = None, sink: torch.Tensor | None = None,
                  softcap: float | None = None, scale: float | None = None, max_len: int = 0, splits: int = 0,
                  out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's newest tokens over its 4-bit pages, bf16 of
    q's shape.

    q: bf16 [B, H, D], or [B, T, H, D] for the T newest tokens (appended before
    the call: token t is position seq_lens - T + t and sees the positions up to
    itself), roped and normed, of any strides that keep its rows 16-byte aligned;
    H a multiple of the pool's K/V heads (head h reads K/V head h // (H / Hkv)).
    n_new: int32 [B], of a padded batch: the first n_new[b] tokens of q are
    sequence b's newest, token t at position seq_lens - n_new + t, and later ones
    get 0 (a count past T is T).  pool, block_table: as ``ops.fp4_quant_append`` wrote them; seq_lens:
    int32 [B].  window: only the newest ``window`` positions up to itself (None:
    all); sink: fp32 [H] or None; softcap: c*tanh(s/c) of the scores, or None;
    scale: of the scores (None: 1/sqrt(D)).  A token that sees nothing gets 0.
    max_len: a bound on seq_lens (0: what the table holds; longer ones are still
    right), which saves short sequences the launch that joins parts of long ones;
    splits: at most about that many workgroups for a K/V head of every sequence,
    instead of as many as the device holds (0).  Up to 64 query rows of a K/V head
    (its query heads times the query tokens; 32 of 129 to 256 dims, any number of
    more dims) the softmax's weights keep 16 bits for the product with the values,
    beyond them 8, as the output has.
    workspace: a tensor of at least ``fp4_attention_workspace`` bytes, of no other
    call that may run at the same time (None: one is allocated for the call)."""
    d, out = _desc(q, pool, block_table, seq_lens, n_new, window, sink, softcap, scale, max_len, splits, out)
    need = int(_lib.load().skv_fp4_attention_workspace(ctypes.byref(d)))
    if need < 0:
        _lib.check(_lib.SKV_EINVAL, "skv_fp4_attention_workspace")
    ws_ptr, ws_bytes = None, 0
    if workspace is not None:
        ws_bytes = workspace.numel() * workspace.element_size()
        if workspace.device != q.device or ws_bytes < need:
            raise ValueError(f"workspace must hold {need} bytes on {q.device}")
        if not workspace.is_contiguous() or workspace.data_ptr() % 16:
            raise ValueError("workspace must be a contiguous tensor whose data is 16-byte aligned")
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        ws_bytes = need
    if workspace is not None:
        ws_ptr = workspace.data_ptr()
    _launch(q.device, "skv_fp4_attention", ctypes.byref(d), ws_ptr, ws_bytes)
    return out


def fp4_attention_workspace(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, *,
                            window: int | None = None, max_len: int = 0, splits: int = 0) -> int:
    """Bytes of workspace that ``fp4_attention`` needs for these shapes (0: none)."""
    lens = torch.empty(q.shape[0], dtype=torch.int32, device=q.device)
    d, _ = _desc(q, pool, block_table, lens, None, window, None, None, None, max_len, splits, None)
    need = int(_lib.load().skv_fp4_attention_workspace(ctypes.byref(d)))
    if need < 0:
        _lib.check(_lib.SKV_EINVAL, "skv_fp4_attention_workspace")
    return need


def _desc(q, pool, block_table, seq_lens, n_new, window, sink, softcap, scale, max_len, splits,
          out) -> tuple[Fp4AttentionDesc, torch.Tensor]:
    _check_layout()
    _require_gpu(q, "q")
    if q.dtype != torch.bfloat16 or q.dim() not in (3, 4):
        raise ValueError(f"q must be bf16 [B, H, D] or [B, T, H, D]; got {q.dtype} {tuple(q.shape)}")
    cache = ops.fp4_cache(pool, block_table)
    kv_heads, shape = cache.n_kv_heads, q.shape
    batch, heads, dim = shape[0], shape[-2], shape[-1]
    if batch != block_table.shape[0] or dim != cache.head_dim:
        raise ValueError(f"q must have {cache.batch} sequences of head_dim {cache.head_dim}; got {tuple(shape)}")
    if heads < 1 or heads % kv_heads:
        raise ValueError(f"q's {heads} heads are not a multiple of the pool's {kv_heads}")
    _require_i32(seq_lens, "seq_lens", (batch,))
    if n_new is not None:
        _require_i32(n_new, "n_new", (batch,))
    if window is not None and window < 1:
        raise ValueError(f"window must be positive (or None); got {window}")
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive (or None); got {softcap}")
    if scale is not None and not scale > 0:
        raise ValueError(f"scale must be positive (or None); got {scale}")
    for name, x in (("scale", scale), ("softcap", softcap)):
        if x is not None and ctypes.c_float(x).value == 0:  # would stand for the default
            raise ValueError(f"{name}={x} is zero in fp32")
    if sink is not None:
        _require_gpu(sink, "sink")
        if sink.dtype != torch.float32 or tuple(sink.shape) != (heads,) or not sink.is_contiguous():
            raise ValueError(f"sink must be a contiguous fp32 [{heads}] tensor")
    strides, data, tokens = q.stride(), q.data_ptr(), shape[1] if len(shape) == 4 else 1
    seq = 2 * strides[0] if batch > 1 else 0
    tok = 2 * strides[1] if tokens > 1 else 0
    head = 2 * strides[-2] if heads > 1 else 0
    if tokens < 1 or strides[-1] != 1 or (data | seq | tok | head) & 15:
        raise ValueError("q needs at least one token, contiguous dims and 16-byte aligned rows")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != torch.bfloat16 or out.shape != shape or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous bf16 {list(shape)} tensor, 16-byte aligned")
    _same_device(q, "q", pool=pool, seq_lens=seq_lens, n_new=n_new, sink=sink, out=out)
    d = Fp4AttentionDesc(cache, seq_lens.data_ptr(), _lib.ptr(n_new), tokens, heads, data, seq, tok, head, out.data_ptr(),
                         _lib.ptr(sink), window or 0, int(max_len), int(splits), scale or 0.0, softcap or 0.0)
    return d, out


class Fp4TokenCache:
    """Paged 4-bit keys and values of ``batch`` ragged sequences for a stack of
    layers that share one block table.

    A step reserves its tokens once and then goes through the layers, each of
    which appends its keys and values and attends:

        cache.reserve(1)
        for i in range(layers):
            cache.append(i, k, v)                # bf16 or fp32 [B, T, Hkv, D]
            out = cache.attention(i, q)          # bf16 [B, T, H, D]

    A prompt goes the same way with its tokens (``n_new`` per sequence where
    they are ragged).  Lengths and free pages are counted on the host, so that a
    reservation or a fork that cannot be raises before it changes anything; steps
    and forks need no synchronisation, a release reads back what it freed.  Up to
    16 layers: a model of more has a cache, with a table of its own, for every 16.
    The pages hold a sequence's whole history, a windowed layer's too.
    """

    def __init__(self, layers: int, batch: int, max_len: int, n_kv_heads: int, head_dim: int, *, block_size: int = 64,
                 n_pages: int | None = None, device: torch.device | str | None = None,
                 page_order_seed: int | None = 0) -> None:
        if not 0 < layers <= MAX_LAYERS:
            raise ValueError(f"1..{MAX_LAYERS} layers supported; got {layers}")
        if not 0 < batch <= MAX_BATCH:
            raise ValueError(f"batch must be in [1, {MAX_BATCH}]; got {batch}")
        if max_len <= 0:
            raise ValueError(f"max_len must be positive; got {max_len}")
        width = -(-max_len // block_size) if block_size > 0 else 1
        pages = batch * width if n_pages is None else n_pages
        # what the calls on it take: tokens of a sequence, pages that a compaction counts, table entries
        if width * block_size > 1 << 24:
            raise ValueError(f"a sequence holds at most 2^24 tokens; got max_len={max_len}")
        if not 0 < pages < 1 << 24:
            raise ValueError(f"n_pages must be in [1, 2^24); got {pages}")
        if batch * (width + 64) > 1 << 30:
            raise ValueError(f"a table of {batch} x {width} pages is too large")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("Fp4TokenCache runs only on a ROCm GPU (no CPU fallback)")
        _lib.load()
        self.device, self.batch, self.max_len, self.block_size = dev, batch, max_len, block_size
        self.n_pages = pages
        self.pool = [ops.fp4_pool(self.n_pages, block_size, n_kv_heads, head_dim, dev) for _ in range(layers)]
        i32 = dict(dtype=torch.int32, device=dev)
        self.block_table = torch.full((batch, width), -1, **i32)
        self.seq_lens = torch.zeros(batch, **i32)
        self.refs = torch.zeros(self.n_pages, **i32)
        self.free_stack, self.free_top = torch.empty(self.n_pages, **i32), torch.empty(1, **i32)
        order = None
        if page_order_seed is not None:
            order = torch.as_tensor(np.random.default_rng(page_order_seed).permutation(self.n_pages).astype(np.int32),
                                    device=dev)
        ops.free_stack_init(self.free_stack, self.free_top, order)
        self.status = torch.zeros(1, **i32)
        # the calls' status words, in turn: a call that succeeds clears its word, which must not be
        # that of one whose refusal nobody has read
        self._words = torch.zeros(STATUS_WORDS, **i32)
        self._word_views = list(self._words.split(1))
        self._word, self._refusals = 0, torch.zeros(STATUS_WORDS, **i32)
        self.host_lens, self.host_free = np.zeros(batch, dtype=np.int64), self.n_pages
        self._n_new: int | torch.Tensor = 0
        self._host_new = np.zeros(batch, dtype=np.int64)  # each sequence's tokens reserved last
        self._most_new, self._padded = 0, False
        self._unwritten: set[int] = set()  # layers that these have not been appended to
        self._recorded: set[int] = set()  # layers that a graph appends to
        self._shared = False  # some of these lie in shared pages
        self._compact_ws = torch.zeros(3 * self.n_pages, **i32)
        self._compact_info = torch.zeros(2, **i32)

    # ----------------------------------------------------------------- step --
    def reserve(self, n_new: int | np.ndarray) -> None:
        """Pages for the next ``n_new`` tokens (one count, or one per sequence) of
        every sequence; the lengths count them from here on."""
        counts = np.broadcast_to(np.asarray(n_new, dtype=np.int64), (self.batch,))
        if (counts < 0).any():
            raise ValueError("n_new must be >= 0")
        if (self.host_lens + counts > self.max_len).any():
            raise RuntimeError(f"Fp4TokenCache overflow: a sequence would exceed max_len={self.max_len}")
        bs = self.block_size
        need = int(((self.host_lens + counts + bs - 1) // bs - (self.host_lens + bs - 1) // bs).sum())
        self._take_pages(need)
        self._n_new = int(n_new) if np.ndim(n_new) == 0 else torch.as_tensor(counts.astype(np.int32),
                                                                            device=self.device)
        ops.reserve(self.free_stack, self.free_top, self.block_table, self.seq_lens, self._n_new, self.block_size,
                    self._status_word())
        self.host_lens = self.host_lens + counts
        self._host_new, self._most_new = counts.copy(), int(counts.max())
        self._shared = self._padded = False
        self._unwritten = set(range(len(self.pool))) if counts.any() else set()

    def _status_word(self) -> torch.Tensor:
        if self._word == STATUS_WORDS:  # all used: what they hold is kept aside
            self._refusals.bitwise_or_(self._words)
            self._word = 0
        self._word += 1
        return self._word_views[self._word - 1]

    def _take_pages(self, need: int) -> None:
        if need > self.host_free:
            raise RuntimeError(f"Fp4TokenCache out of pages: {need} needed, {self.host_free} free")
        self.host_free -= need

    def append(self, i: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Layer i's keys and values [B, T, Hkv, D] of the tokens reserved last
        (of sequence b the first n_new[b], T at least the largest of them); not after a
        fork of these, which lie in shared pages then."""
        if k.dim() == 4 and k.shape[1] < self._most_new:
            raise ValueError(f"{self._most_new} tokens of a sequence were reserved, k has {k.shape[1]}")
        if self._shared:
            raise RuntimeError("the tokens reserved last are a fork's, too; reserve new ones to append")
        ops.fp4_quant_append(self.pool[i], self.block_table, self.seq_lens, k, v, self._n_new)
        self._padded = k.shape[1] > self._most_new
        layer = range(len(self.pool))[i]
        self._unwritten.discard(layer)
        if torch.cuda.is_current_stream_capturing():
            self._recorded.add(layer)

    def attention(self, i: int, q: torch.Tensor, *, window: int | None = None, sink: torch.Tensor | None = None,
                  softcap: float | None = None, scale: float | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
        """``fp4_attention`` of layer i for the queries of the newest tokens; after a
        ragged reservation of sequence b's first n_new[b] (the others get 0)."""
        n_new = self._n_new if isinstance(self._n_new, torch.Tensor) else None
        if n_new is None and self._padded and q.dim() == 4 and q.shape[1] > self._n_new:
            # the newest of several reservations, or a padded batch as k and v were
            raise ValueError(f"{self._n_new} tokens were reserved, q has {q.shape[1]}: reserve a count for each sequence "
                             "for a padded batch")
        return fp4_attention(q, self.pool[i], self.block_table, self.seq_lens, n_new=n_new, window=window, sink=sink,
                             softcap=softcap, scale=scale, max_len=int(self.host_lens.max()), out=out)

    def check_status(self) -> None:
        """Synchronise and raise if the device refused a reservation, fork or release
        since the last check, as it does where the tables were changed behind the
        host's back (it wrote nothing; the host's counts are read back)."""
        bits = int(np.bitwise_or.reduce(torch.cat((self._refusals, self._words, self.status)).cpu().numpy()))
        if bits:
            for t in (self._refusals, self._words, self.status):
                t.zero_()
            self.host_lens = self.seq_lens.cpu().numpy().astype(np.int64)
            self.host_free = int(self.free_top.item())
            raise RuntimeError(f"Fp4TokenCache reservation, fork or release refused (status bits {bits})")

    # ------------------------------------------------------ forks, eviction --
    def fork(self, src: list[int], dst: list[int]) -> None:
        """Make the empty sequences dst[f] copies of src[f], sharing their whole
        pages; raises (and changes nothing) if the pool lacks a page for a begun one, or
        a layer still has to append the tokens that a source reserved last (layers whose
        append a graph replays are taken to have done so)."""
        src, dst = check_forks(src, dst, self.host_lens)
        if not len(src):
            return
        newest = self._host_new[src]
        missing = self._unwritten - self._recorded
        if newest.any() and missing:
            raise RuntimeError(f"a fork's source has reserved tokens that have not been appended to layers {sorted(missing)}")
        self._take_pages(int((self.host_lens[src] % self.block_size != 0).sum()))
        idx = torch.as_tensor(np.stack([src, dst]).astype(np.int32), device=self.device)
        ops.fork(self.free_stack, self.free_top, self.refs, self.block_table, self.seq_lens, idx[0], idx[1],
                 self.block_size, self.pool, self._status_word())
        self.host_lens[dst] = self.host_lens[src]
        if isinstance(self._n_new, torch.Tensor):  # the newest tokens of a copy are its source's
            ops.copy_slots([self._n_new], idx[0], idx[1])
        self._host_new[dst] = newest
        self._shared |= bool(newest.any())

    def release(self, mask: np.ndarray) -> None:
        """Finish the sequences with mask[b]: the pages that no other sequence holds
        return to the free list."""
        mask = np.asarray(mask, dtype=bool)
        if mask.shape != (self.batch,):
            raise ValueError("mask must be [batch]")
        if (mask & (self.host_lens == 0)).any():
            raise RuntimeError("release of a sequence that holds no tokens (double free)")
        ops.release(self.free_stack, self.free_top, self.block_table, self.seq_lens,
                    torch.as_tensor(mask.astype(np.uint8), device=self.device), self.block_size, self._status_word(),
                    refs=self.refs)
        self._host_new[mask] = 0
        self.check_status()
        self.host_lens[mask] = 0
        self.host_free = int(self.free_top.item())

    def compact(self) -> tuple[int, int]:
        """Defragment the pages; returns (n_live, n_moved)."""
        ops.compact(self.pool, self.block_table, self.seq_lens, self.block_size, self.free_stack, self.free_top,
                    self._compact_ws, self._compact_info, refs=self.refs)
        live, moved = self._compact_info.cpu().tolist()
        return live, moved


def check_forks(src, dst, host_lens: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """The sequences of a fork as arrays, or the error of forks that cannot be.  Copies of
    an empty sequence are left out: a destination is empty already, and one that is
    another fork's source too would be read while it is written."""
    src, dst = np.atleast_1d(np.asarray(src, dtype=np.int64)), np.atleast_1d(np.asarray(dst, dtype=np.int64))
    if src.ndim != 1 or src.shape != dst.shape:
        raise ValueError("src and dst must name as many sequences")
    for x in (src, dst):
        if ((x < 0) | (x >= host_lens.shape[0])).any():
            raise ValueError(f"sequences must be in [0, {host_lens.shape[0]})")
    if np.unique(dst).size != dst.size:
        raise ValueError("a sequence cannot be forked to twice")
    if (host_lens[dst] != 0).any():
        raise RuntimeError("a fork needs empty sequences to go to; release them first")
    held = host_lens[src] != 0
    return src[held], dst[held]
