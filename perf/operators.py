"""The operators of a token cache held in 4 bits and of pages that sequences share, as timed cases.

Three kinds of call, each through the public Python API:

* ``write``  : new tokens' keys and values go into the 4-bit pages (``ops.fp4_quant_append``) and come back as the
  values that the pages now hold (``ops.fp4_gather``).
* ``attend`` : attention of one or more query tokens per sequence over the 4-bit pages (``fp4_attention``).
* ``fork``   : sequences are forked onto shared pages (``ops.fork``), some are freed (``ops.release`` with reference
  counts) and, where a case says so, the pages are compacted (``ops.compact`` with reference counts).

A page of the 4-bit cache holds ``block`` tokens of every K/V head.  Per head: the keys' codes (two dims a byte, the
even dim in the low half), the values' codes, then per token a scale byte for each 32 dims of the key, then of the
value.  A code is e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), a scale byte s stands for 2^(s - 127).

Sizes are those of the repository's benchmark and tests where it has them (contexts of 1k to 1M tokens, heads of 64 x
128 and 512 dims, windows of 128, pages of 16 and 64 tokens, rows of 576 dims), generic ones elsewhere.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

BF, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _dev() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _api():
    pkg = str(Path(__file__).resolve().parents[1] / "saint-llm_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import saint_kv

    return saint_kv


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # a decode step's write: one token of every sequence into its page, read back for a check of the cache
        {"name": "write_step", "kind": "write", "batch": 64, "lmin": 1024, "lmax": 4096, "t_new": 1, "kv_heads": 8,
         "dim": 128, "block": 64, "f32": False, "spread": 1},
        # prompts of 8k tokens enter the cache whole
        {"name": "write_prompt", "kind": "write", "batch": 8, "lmin": 8192, "lmax": 8192, "t_new": 8192, "kv_heads": 8,
         "dim": 128, "block": 64, "f32": False, "spread": 2},
        # ragged chunks of an fp32 model with an odd number of heads, in pages of 16
        {"name": "write_ragged", "kind": "write", "batch": 5, "lmin": 700, "lmax": 2500, "t_new": 611, "kv_heads": 3,
         "dim": 96, "block": 16, "f32": True, "spread": 3},
        # the first tokens of a chat: one short sequence, where only latency counts
        {"name": "attend_one", "kind": "attend", "batch": 1, "lmin": 333, "lmax": 333, "t_new": 1, "heads": 16,
         "kv_heads": 2, "dim": 128, "block": 16, "window": 0, "sink": False, "softcap": 0.0, "spread": 4},
        # a serving batch's decode step, 8 query heads to a K/V head, ragged 1k - 32k contexts
        {"name": "attend_step", "kind": "attend", "batch": 64, "lmin": 1024, "lmax": 32768, "t_new": 1, "heads": 64,
         "kv_heads": 8, "dim": 128, "block": 64, "window": 0, "sink": False, "softcap": 0.0, "spread": 5},
        # the same with all 64 heads on one K/V head, contexts of 64k
        {"name": "attend_mqa_64k", "kind": "attend", "batch": 16, "lmin": 65536, "lmax": 65536, "t_new": 1, "heads": 64,
         "kv_heads": 1, "dim": 128, "block": 64, "window": 0, "sink": True, "softcap": 0.0, "spread": 6},
        # few long requests: 256k - 1M tokens, four drafted tokens checked at once
        {"name": "attend_1m", "kind": "attend", "batch": 4, "lmin": 262144, "lmax": 1048576, "t_new": 4, "heads": 16,
         "kv_heads": 4, "dim": 64, "block": 64, "window": 0, "sink": False, "softcap": 0.0, "spread": 7},
        # a sliding-window layer's step: 128 tokens of wide heads, sink and softcap
        {"name": "attend_window", "kind": "attend", "batch": 32, "lmin": 100, "lmax": 8192, "t_new": 1, "heads": 64,
         "kv_heads": 1, "dim": 512, "block": 16, "window": 128, "sink": True, "softcap": 30.0, "spread": 8},
        # a prompt's chunk over what the cache holds of it, itself included
        {"name": "attend_chunk", "kind": "attend", "batch": 2, "lmin": 16001, "lmax": 16384, "t_new": 1000, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 64, "window": 0, "sink": False, "softcap": 0.0, "spread": 9},
        # one more answer to a short prompt
        {"name": "fork_one", "kind": "fork", "batch": 2, "forks": 1, "sources": 1, "lmin": 333, "lmax": 333,
         "kv_heads": 2, "dim": 128, "block": 16, "pools": 1, "compact": False, "spread": 10},
        # several answers to each of a batch of long prompts, in a cache of eight layers, freed again
        {"name": "fork_samples", "kind": "fork", "batch": 64, "forks": 48, "sources": 16, "lmin": 8192, "lmax": 65536,
         "kv_heads": 1, "dim": 512, "block": 64, "pools": 8, "compact": False, "spread": 11},
        # the same where a third of the prompts is done: they leave, and what is live is moved together
        {"name": "fork_compact", "kind": "fork", "batch": 48, "forks": 24, "sources": 24, "lmin": 4096, "lmax": 32768,
         "kv_heads": 1, "dim": 512, "block": 64, "pools": 2, "compact": True, "spread": 12},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the listed ranges."""
    while True:
        kind = rng.choice(["write", "attend", "attend", "attend", "fork"])
        block = rng.choice([16, 32, 64, 64, 128])
        dim = rng.choice([32, 64, 64, 96, 128, 128, 160, 256, 512])
        if kind == "write":
            t = rng.choice([1, _log(rng, 2, 8192)])
            c = {"batch": _log(rng, 1, 64), "lmin": t, "lmax": max(t, _log(rng, t, 16384)), "t_new": t,
                 "kv_heads": rng.choice([1, 2, 3, 8]), "dim": dim, "block": block, "f32": rng.random() < 0.3}
            c.update(kind=kind, spread=rng.randrange(1 << 30))
            fits = _write_values(c) <= 2 ** 27 and _pages(c) * block * c["kv_heads"] * dim <= 2 ** 30
        elif kind == "attend":
            t = rng.choice([1, 1, _log(rng, 2, 1000)])
            top = _log(rng, max(8, t), 524288 if t < 8 else 16384)
            kv = rng.choice([1, 1, 2, 4, 8])
            c = {"batch": _log(rng, 1, 64), "lmin": max(1, int(top * rng.uniform(0.05, 1.0))), "lmax": top, "t_new": t,
                 "heads": kv * rng.choice([1, 3, 4, 8, 16]), "kv_heads": kv, "dim": dim, "block": block,
                 "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "sink": rng.random() < 0.4,
                 "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
            c.update(kind=kind, spread=rng.randrange(1 << 30))
            padded = c["batch"] * c["lmax"]
            fits = (padded * kv * dim <= 2 ** 31 and padded * c["heads"] * t <= 2 ** 30
                    and padded * c["heads"] * t * dim <= 2 ** 37)
        else:
            n = _log(rng, 1, 24)
            c = {"batch": 2 * n + rng.randint(0, 8), "forks": rng.randint(1, n), "sources": n,
                 "lmin": _log(rng, 1, 8192), "lmax": 0, "kv_heads": rng.choice([1, 2, 8]), "dim": dim, "block": block,
                 "pools": rng.randint(1, 8), "compact": rng.random() < 0.3}
            c["lmax"] = _log(rng, c["lmin"], 65536)
            c.update(kind=kind, spread=rng.randrange(1 << 30))
            fits = 2 * _pages(c) * block * c["kv_heads"] * dim * c["pools"] <= 2 ** 32
        if fits:
            return c


def _lens(c: dict, n: int) -> list[int]:
    """The lengths of n sequences, spread over the logarithm; in larger batches one is empty or as short as it can be."""
    r = random.Random(c["spread"])
    got = [_log(r, c["lmin"], c["lmax"]) for _ in range(n)]
    if c["kind"] == "attend" and n > 8 and c["lmin"] < 2048:
        got[r.randrange(n)] = r.choice([0, 1])
    return got


def _new(c: dict, lens: list[int]) -> list[int]:
    """New tokens of each sequence of a write: all of t_new, or of a larger ragged batch fewer, in one sequence none."""
    r = random.Random(c["spread"] + 1)
    got = [min(c["t_new"], n) for n in lens]
    if c["t_new"] > 1 and c["lmin"] < c["lmax"]:
        got = [r.randint(1, n) for n in got]
        if len(got) > 4:
            got[r.randrange(len(got))] = 0
    return got


def _pages(c: dict) -> int:
    n = c["sources"] if c["kind"] == "fork" else c["batch"]
    return sum(-(-x // c["block"]) for x in _lens(c, n))


def _write_values(c: dict) -> int:
    return 2 * c["batch"] * c["t_new"] * c["kv_heads"] * c["dim"]


def _row_bytes(c: dict) -> int:
    return c["kv_heads"] * c["dim"] * 17 // 16  # K and V of a token: codes and scales


def _pairs(c: dict) -> int:
    """(query token, token that it sees) pairs of all sequences."""
    got = 0
    for n in _lens(c, c["batch"]):
        for t in range(c["t_new"]):
            see = max(0, n - c["t_new"] + t + 1)
            got += min(see, c["window"]) if c["window"] else see
    return got


def work(c: dict) -> dict:
    if c["kind"] == "write":
        n = sum(_new(c, _lens(c, c["batch"])))
        values = 2 * n * c["kv_heads"] * c["dim"]
        # source read, codes and scales written and read, bf16 values written
        return {"bytes": values * ((4 if c["f32"] else 2) + 2) + 2 * n * _row_bytes(c), "flops": 0}
    if c["kind"] == "attend":
        seen = 0
        for n in _lens(c, c["batch"]):
            seen += min(n, c["window"] + c["t_new"] - 1) if c["window"] else n
        q = c["batch"] * c["t_new"] * c["heads"] * c["dim"]
        return {"bytes": seen * _row_bytes(c) + 4 * q, "flops": 4 * _pairs(c) * c["heads"] * c["dim"]}
    lens = _lens(c, c["sources"])
    page = c["block"] * _row_bytes(c) * c["pools"]
    src, dst, gone = _fork_plan(c)
    copied = sum(1 for s in src if lens[s] % c["block"])
    tables = sum(-(-lens[s] // c["block"]) for s in src) * 4
    got = 2 * copied * page + 6 * tables  # rows copied; table read and written, counts up, read for the release, down
    if c["compact"]:
        got += 2 * page * _moved(c)
    return {"bytes": max(got, 64), "flops": 0}


def _fork_plan(c: dict) -> tuple[list[int], list[int], list[int]]:
    """Sources and destinations of the forks, and the sequences that leave afterwards: the forks, or with compaction a
    third of the sources (whose pages live on in their forks) and the pages between."""
    r = random.Random(c["spread"] + 2)
    src = [r.randrange(c["sources"]) for _ in range(c["forks"])]
    dst = r.sample(range(c["sources"], c["batch"]), c["forks"])
    gone = sorted(r.sample(range(c["sources"]), max(1, c["sources"] // 3))) if c["compact"] else dst
    return src, dst, gone


def _moved(c: dict) -> int:
    """Pages that the compaction moves, about: live ones at or past the number of live ones."""
    lens = _lens(c, c["sources"])
    src, _, gone = _fork_plan(c)
    pages = [-(-n // c["block"]) for n in lens]
    keep = sum(p if i not in gone else (lens[i] // c["block"] if i in src else 0) for i, p in enumerate(pages))
    keep += sum(1 for s in src if lens[s] % c["block"])
    total = sum(pages) + c["forks"]
    return int(keep * (1 - keep / max(total, 1)))


# ---------------------------------------------------------------------------
# The 4-bit format in elementary operations
# ---------------------------------------------------------------------------
def _pow2(e: torch.Tensor) -> torch.Tensor:
    return ((e.int() + 127) << 23).view(F32)


def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (packed two a byte) and scale bytes of x [..., D]: per 32 dims the smallest power of two under which no
    value passes 6, each value rounded to the nearest level (ties to the even code)."""
    b = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(m > 0.75, e - 2, e - 3).clamp(-120, 125)
    e = torch.where(m == 0, torch.full_like(e, -120), e)
    a = b * _pow2(-e).unsqueeze(-1)
    sign = torch.signbit(a)
    a = a.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5.0).byte())
    code = (code + 8 * sign.byte()).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], (e + 127).byte()


def _dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """[..., D / 2] bytes and [..., D / 32] scale bytes to values [..., D]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    both = torch.stack([level.repeat(16), level.repeat_interleave(16)], -1)  # of every byte: low, high
    v = both.index_select(0, codes.flatten().int()).view(*codes.shape[:-1], scales.shape[-1], 32)
    return (v * _pow2(scales.int() - 127).unsqueeze(-1)).flatten(-2)


def _planes(pool: torch.Tensor, block: int, dim: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Views of the pages: key codes, value codes [P, Hkv, block, D / 2], scale bytes [P, Hkv, block, 2, D / 32]."""
    heads = pool.shape[2]
    flat = pool.view(pool.shape[0], heads, -1)
    half = block * dim // 2
    return (flat[..., :half].unflatten(-1, (block, -1)), flat[..., half:2 * half].unflatten(-1, (block, -1)),
            flat[..., 2 * half:].unflatten(-1, (block, 2, -1)))


def _pool(c: dict, n_pages: int) -> torch.Tensor:
    return torch.zeros(n_pages, c["block"], c["kv_heads"], c["dim"] * 17 // 16, dtype=torch.uint8, device=_dev())


def _tables(c: dict, seed: int, lens: list[int], batch: int, n_pages: int) -> tuple[torch.Tensor, list[int]]:
    """A block table over a random permutation of the pages, and the ids that are left, in the order of their use."""
    order = list(range(n_pages))
    random.Random(seed).shuffle(order)
    width = max(1, max(-(-n // c["block"]) for n in lens))
    bt = torch.full((batch, width), -1, dtype=I32)
    at = 0
    for b, n in enumerate(lens):
        p = -(-n // c["block"])
        bt[b, :p] = torch.tensor(order[at:at + p], dtype=I32)
        at += p
    return bt.to(_dev()), order[at:]


def _fill(c: dict, pool: torch.Tensor, gen: torch.Generator) -> None:
    """Every page of normally distributed keys and values, as after prompts."""
    kc, vc, sc = _planes(pool, c["block"], c["dim"])
    step = max(1, 2 ** 27 // (c["block"] * c["kv_heads"] * c["dim"]))
    for p in range(0, pool.shape[0], step):
        n = min(step, pool.shape[0] - p)
        for i, codes in enumerate((kc, vc)):
            x = torch.randn(n, c["kv_heads"], c["block"], c["dim"], generator=gen, device=pool.device)
            codes[p:p + n], sc[p:p + n, :, :, i] = _quantize(x)


# ---------------------------------------------------------------------------
# States
# ---------------------------------------------------------------------------
def prepare(c: dict, seed: int) -> dict:
    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "fork":
        return _prepare_fork(c, seed, gen, s)
    lens = _lens(c, c["batch"])
    n_pages = sum(-(-n // c["block"]) for n in lens) + 3
    s["pool"] = _pool(c, n_pages)
    s["bt"], _ = _tables(c, seed, lens, c["batch"], n_pages)
    s["lens"] = torch.tensor(lens, dtype=I32, device=dev)
    if c["kind"] == "write":
        new = _new(c, lens)
        s["n_new"] = torch.tensor(new, dtype=I32, device=dev)
        # keys and values side by side, as one projection writes them; a few channels are far larger than the rest
        kv = torch.randn(c["batch"], c["t_new"], 2, c["kv_heads"], c["dim"], generator=gen, device=dev)
        kv *= torch.where(torch.rand(c["kv_heads"], c["dim"], generator=gen, device=dev) < 0.02, 20.0, 1.0)
        kv = kv if c["f32"] else kv.to(BF)
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        shape = (c["batch"], c["t_new"], c["kv_heads"], c["dim"])
        s["out_k"], s["out_v"] = torch.zeros(shape, dtype=BF, device=dev), torch.zeros(shape, dtype=BF, device=dev)
        return s
    _fill(c, s["pool"], gen)
    s["q"] = torch.randn(c["batch"], c["t_new"], c["heads"], c["dim"], generator=gen, device=dev).to(BF)
    s["sink"] = torch.randn(c["heads"], generator=gen, device=dev) if c["sink"] else None
    s["max_len"] = max(1, max(lens))
    return s


def _prepare_fork(c: dict, seed: int, gen: torch.Generator, s: dict) -> dict:
    dev = _dev()
    lens = _lens(c, c["sources"]) + [0] * (c["batch"] - c["sources"])
    used = sum(-(-n // c["block"]) for n in lens)
    n_pages = used + c["forks"] + 3
    bt, free = _tables(c, seed, lens, c["batch"], n_pages)
    # tables, lengths, counts and the free stack in one buffer: a pass starts from the kept copy of it
    parts = [bt.flatten(), torch.tensor(lens, dtype=I32, device=dev), torch.zeros(n_pages, dtype=I32, device=dev),
             torch.tensor(free[::-1] + [0] * (n_pages - len(free)), dtype=I32, device=dev),
             torch.tensor([len(free)], dtype=I32, device=dev), torch.zeros(4, dtype=I32, device=dev)]
    sizes = [-(-p.numel() // 4) * 4 for p in parts]
    s["kept"] = torch.cat([torch.nn.functional.pad(p, (0, n - p.numel())) for p, n in zip(parts, sizes)])
    s["books"] = s["kept"].clone()
    views = s["books"].split(sizes)
    s["bt"] = views[0][:bt.numel()].view(bt.shape)
    for name, v, p in zip(("lens", "refs", "stack", "top", "status"), views[1:], parts[1:]):
        s[name] = v[:p.numel()]
    s["status"], s["info"] = s["status"][:1], s["status"][2:4]
    src, dst, gone = _fork_plan(c)
    s["src"], s["dst"] = torch.tensor(src, dtype=I32, device=dev), torch.tensor(dst, dtype=I32, device=dev)
    s["gone"] = torch.zeros(c["batch"], dtype=torch.bool, device=dev)
    s["gone"][torch.tensor(gone, device=dev)] = True
    s["pools"] = []
    for _ in range(c["pools"]):
        pool = _pool(c, n_pages)
        pool.view(-1).view(I64).random_(generator=gen)  # a page is whole blocks of 16 tokens
        s["pools"].append(pool)
    if c["compact"]:
        s["ws"] = torch.zeros(3 * n_pages, dtype=I32, device=dev)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s: dict):
    c = s["case"]
    if own:
        kv = _api()
        if c["kind"] == "write":
            kv.ops.fp4_quant_append(s["pool"], s["bt"], s["lens"], s["k"], s["v"], s["n_new"])
            kv.ops.fp4_gather(s["pool"], s["bt"], s["lens"], s["out_k"], s["out_v"], s["n_new"])
            return s["out_k"], s["out_v"]
        if c["kind"] == "attend":
            return kv.fp4_attention(s["q"], s["pool"], s["bt"], s["lens"], window=c["window"] or None, sink=s["sink"],
                                    softcap=c["softcap"] or None, max_len=s["max_len"])
        s["books"].copy_(s["kept"])
        kv.ops.fork(s["stack"], s["top"], s["refs"], s["bt"], s["lens"], s["src"], s["dst"], c["block"], s["pools"],
                    s["status"])
        kv.ops.release(s["stack"], s["top"], s["bt"], s["lens"], s["gone"], c["block"], s["status"], refs=s["refs"])
        if c["compact"]:
            kv.ops.compact(s["pools"], s["bt"], s["lens"], c["block"], s["stack"], s["top"], s["ws"], s["info"],
                           refs=s["refs"])
        return [s["books"], *s["pools"]]
    if c["kind"] == "write":
        return _plain_write(s)
    if c["kind"] == "attend":
        return _plain_attend(s)
    s["books"].copy_(s["kept"])
    _plain_fork(s)
    _plain_release(s)
    if c["compact"]:
        _plain_compact(s)
    return [s["books"], *s["pools"]]


def _plain_write(s: dict):
    c = s["case"]
    t = torch.arange(c["t_new"], device=s["lens"].device)
    live = t[None] < s["n_new"][:, None]
    at = (s["lens"] - s["n_new"])[:, None] + t[None]
    b, i = live.nonzero(as_tuple=True)
    pos = at[b, i]
    page, slot = s["bt"][b, pos // c["block"]].long(), (pos % c["block"]).long()
    kc, vc, sc = _planes(s["pool"], c["block"], c["dim"])
    for j, (x, codes, out) in enumerate(((s["k"], kc, s["out_k"]), (s["v"], vc, s["out_v"]))):
        q, e = _quantize(x[b, i])
        codes[page, :, slot] = q
        sc[page, :, slot, j] = e
        out[b, i] = _dequantize(codes[page, :, slot], sc[page, :, slot, j]).to(BF)
    return s["out_k"], s["out_v"]


def _plain_attend(s: dict) -> torch.Tensor:
    c = s["case"]
    kv, g, d, t = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["t_new"]
    bt = s["bt"].clamp_min(0).long()
    kc, vc, sc = _planes(s["pool"], c["block"], d)
    scales = sc[bt].transpose(1, 2).flatten(2, 3)  # [B, Hkv, L, 2, D / 32]

    def rows(codes, j):
        return _dequantize(codes[bt].transpose(1, 2).flatten(2, 3), scales[:, :, :, j])

    k = rows(kc, 0)
    n = k.shape[2]
    q = s["q"].float().view(-1, t, kv, g, d).permute(0, 2, 3, 1, 4).reshape(-1, kv, g * t, d)
    a = torch.matmul(q, k.transpose(2, 3)).view(-1, kv, g, t, n) / math.sqrt(d)
    del k
    if c["softcap"]:
        a = c["softcap"] * torch.tanh(a / c["softcap"])
    pos = torch.arange(n, device=a.device)
    last = (s["lens"].long()[:, None] - t + torch.arange(t, device=a.device))[:, :, None]
    seen = (pos <= last) & (pos < s["lens"][:, None, None])
    if c["window"]:
        seen &= pos > last - c["window"]
    seen = seen[:, None, None]
    a = a.masked_fill(~seen, -math.inf)
    top = a.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, kv, g, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    a = torch.exp(a - top)
    total = a.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    a = a / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(a.view(-1, kv, g * t, n), rows(vc, 1))
    return out.view(-1, kv, g, t, d).permute(0, 3, 1, 2, 4).reshape(-1, t, kv * g, d).to(BF)


def _plain_fork(s: dict) -> None:
    """Whole pages are shared (their count of further owners goes up), the page that the last tokens begin is copied
    into a page from the free stack, forks in order."""
    block, bt, lens = s["case"]["block"], s["bt"], s["lens"]
    src, dst = s["src"].long(), s["dst"].long()
    n = lens[src].long()
    full, part = n // block, n % block > 0
    row = torch.arange(bt.shape[1], device=bt.device)
    shared = row[None] < full[:, None]
    rows = torch.where(shared, bt[src], bt[dst])
    rank = part.long().cumsum(0)
    fresh = s["stack"][(s["top"].long() - rank).clamp_min(0)]
    at = full.clamp_max(bt.shape[1] - 1)[:, None]
    old = bt[src].gather(1, at)
    rows = torch.where(part[:, None] & (row[None] == at), fresh[:, None], rows)
    s["refs"].index_add_(0, bt[src][shared].long(), torch.ones_like(bt[src][shared]))
    bt[dst] = rows
    lens[dst] = lens[src]
    s["top"].sub_(rank[-1:].to(I32))
    for pool in s["pools"]:
        pool[fresh[part].long()] = pool[old[part, 0].long()]


def _plain_release(s: dict) -> None:
    """Pages whose last owner leaves go on the free stack: sequences ascending, a sequence's pages from its last to its
    first, a page that several of them hold at the last of them."""
    block, bt, lens = s["case"]["block"], s["bt"], s["lens"]
    width = bt.shape[1]
    held = torch.arange(width, device=bt.device)[None] < ((lens + block - 1) // block)[:, None]
    held = held & s["gone"][:, None]
    pages = bt.flip(1)[held.flip(1)].long()  # in the order of release
    n = s["refs"].shape[0]
    leave = torch.zeros(n, dtype=I32, device=bt.device).index_add_(0, pages, torch.ones_like(pages, dtype=I32))
    last = torch.full((n,), -1, dtype=I64, device=bt.device)
    order = torch.arange(pages.shape[0], device=bt.device)
    last.scatter_reduce_(0, pages, order, "amax")
    free = leave == s["refs"] + 1
    push = pages[free[pages] & (last[pages] == order)]
    s["stack"][s["top"].long() + torch.arange(push.shape[0], device=bt.device)] = push.to(I32)
    s["top"].add_(push.shape[0])
    s["refs"].sub_(torch.where(free, s["refs"], leave))
    bt.masked_fill_(held, -1)
    lens.masked_fill_(s["gone"], 0)


def _plain_compact(s: dict) -> None:
    """Live pages at or past the number of live ones move, ascending, into the free ids below it; pops then return the
    ids from there on."""
    block, bt, lens, n = s["case"]["block"], s["bt"], s["lens"], s["refs"].shape[0]
    held = torch.arange(bt.shape[1], device=bt.device)[None] < ((lens + block - 1) // block)[:, None]
    live = torch.zeros(n, dtype=torch.bool, device=bt.device)
    live[bt[held].long()] = True
    ids = torch.arange(n, device=bt.device)
    n_live = live.sum()
    moved, holes = ids[live & (ids >= n_live)], ids[~live & (ids < n_live)]
    to = ids.clone()
    to[moved] = holes
    bt.copy_(torch.where(held, to[bt.clamp_min(0).long()].to(I32), bt))
    for pool in s["pools"]:
        pool[holes] = pool[moved]
    s["refs"][holes] = s["refs"][moved]
    s["refs"][moved] = 0
    rest = ids[n_live:]
    s["stack"][:rest.shape[0]] = rest.flip(0).to(I32)
    s["top"].fill_(rest.shape[0])
    s["info"].copy_(torch.stack([n_live, torch.as_tensor(moved.shape[0], device=bt.device)]).to(I32))


# ---------------------------------------------------------------------------
# In 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_values(nibbles: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """(-1)^sign * 2^(E - 1) * (1 + M / 2), or M / 2 where E = 0, times 2^(scale - 127)."""
    sign, e, m = nibbles // 8, nibbles // 2 % 4, nibbles % 2
    mag = torch.where(e == 0, 0.5 * m.double(), (1 + 0.5 * m.double()) * 2.0 ** (e.double() - 1))
    return (1 - 2 * sign.double()) * mag * 2.0 ** (scale.double() - 127)


def _exact_rows(pool: torch.Tensor, pages: torch.Tensor, head: int, n: int, block: int, dim: int):
    """Keys and values [n, D] of one head of one sequence."""
    flat = pool.view(pool.shape[0], pool.shape[2], -1)[pages.long(), head].long()
    half = block * dim // 2
    scales = flat[:, 2 * half:].reshape(-1, 2, dim // 32)[:n]
    got = []
    for j in range(2):
        code = flat[:, j * half:(j + 1) * half].reshape(-1, dim // 2)[:n]
        nib = torch.stack([code & 15, code >> 4], -1).reshape(-1, dim)
        got.append(_exact_values(nib, scales[:, j].repeat_interleave(32, -1)))
    return got


def exact(c: dict, seed: int):
    if c["kind"] == "fork":
        return None
    s = prepare(c, seed)
    lens = _lens(c, c["batch"])
    if c["kind"] == "write":
        outs = []
        for x in (s["k"], s["v"]):
            out = torch.zeros(x.shape, dtype=F64, device=x.device)
            levels = torch.tensor(LEVELS, dtype=F64, device=x.device)
            mid = (levels[1:] + levels[:-1]) / 2
            for b, n in enumerate(_new(c, lens)):
                v = x[b, :n].double().reshape(n, c["kv_heads"], c["dim"] // 32, 32)
                big = v.abs().amax(-1, keepdim=True).clamp_min(6.0 * 2.0 ** -120)
                scale = ((torch.ceil(torch.log2(big / 6) - 1e-13).long() + 1023) << 52).view(F64)
                a = v.abs() / scale
                code = torch.bucketize(a, mid, right=True)  # ties upwards
                tie = (a == mid[(code - 1).clamp_min(0)]) & (code > 0) & (code % 2 == 1)
                out[b, :n] = (torch.sign(v) * levels[(code - tie.long())] * scale).reshape(n, c["kv_heads"], c["dim"])
            outs.append(out)
        return tuple(outs)
    if 4.0 * _pairs(c) * c["heads"] * c["dim"] > 3e13:
        return None
    t, g = c["t_new"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=F64, device=s["q"].device)
    for b, n in enumerate(lens):
        pages = s["bt"][b, :-(-n // c["block"])]
        first = max(0, t - n)  # query tokens before the sequence's start see nothing
        if n == 0:
            continue
        at = torch.arange(n, device=out.device)
        here = torch.arange(n - t + first, n, device=out.device)[:, None]
        hidden = at[None] > here
        if c["window"]:
            hidden |= at[None] <= here - c["window"]
        for h in range(c["kv_heads"]):
            k, v = _exact_rows(s["pool"], pages, h, n, c["block"], c["dim"])
            for i in range(h * g, (h + 1) * g):
                a = s["q"][b, first:, i].double() @ k.T / math.sqrt(c["dim"])
                if c["softcap"]:
                    a = c["softcap"] * torch.tanh(a / c["softcap"])
                a = a.masked_fill(hidden, -math.inf)
                if s["sink"] is not None:
                    a = torch.cat([a, s["sink"][i].double().expand(a.shape[0], 1)], 1)
                out[b, first:, i] = torch.softmax(a, 1)[:, :n] @ v
    return out
