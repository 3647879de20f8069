"""The operators of drafted tokens, of windows that keep their first tokens, and of token probabilities, as timed cases.

Four kinds of call, each through the public Python API:

* ``tree``   : attention of a tree of drafted tokens over the 4-bit cache (``fp4_attention`` with ``tree``).  A node sees
  the tokens before the drafted ones, its ancestors and itself.
* ``stream`` : attention with a sliding window and a few first tokens that stay visible (``fp4_attention`` with ``window``
  and ``first``), for single tokens and for a prompt's chunk.
* ``score``  : log probabilities of given tokens with the entropy and the most likely alternatives of each row of logits
  (``ops.token_logprobs``).
* ``keep``   : after the model has checked a tree: its masks and depths (``ops.draft_tree``), the accepted path
  (``ops.accept_drafts``), and the accepted tokens moved together in every layer's pages, the lengths cut, the pages
  behind them freed (``ops.keep_tokens``).

A token's history is the tokens before the drafted ones, then those of its mask in their order (without a tree: every
token up to itself); ``window`` and ``first`` count in it.

A page of the 4-bit cache holds ``block`` tokens of every K/V head.  Per head: the keys' codes (two dims a byte, the
even dim in the low half), the values' codes, then per token a scale byte for each 32 dims of the key, then of the
value.  A code is e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), a scale byte s stands for 2^(s - 127).

Sizes are those of the repository's benchmark and tests where it has them (contexts of 1k to 1M tokens, heads of 64 x
128 and 512 dims, windows of 128, pages of 16 and 64 tokens), generic ones elsewhere.
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
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _dev() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _api():
    if "saint_kv" not in sys.modules:  # a program finds and imports it once
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "saint-llm_amd"))
    import saint_kv

    return saint_kv


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # eight drafted tokens of one short chat, where only latency counts
        {"name": "tree_one", "kind": "tree", "batch": 1, "lmin": 341, "lmax": 341, "nodes": 8, "heads": 16,
         "kv_heads": 2, "dim": 128, "block": 16, "window": 0, "first": 0, "sink": False, "softcap": 0.0, "spread": 1},
        # a serving batch's trees of up to 32 nodes, 8 query heads to a K/V head, ragged 1k - 16k contexts
        {"name": "tree_step", "kind": "tree", "batch": 32, "lmin": 1024, "lmax": 16384, "nodes": 32, "heads": 64,
         "kv_heads": 8, "dim": 128, "block": 64, "window": 0, "first": 0, "sink": False, "softcap": 0.0, "spread": 2},
        # small trees of a few long requests
        {"name": "tree_long", "kind": "tree", "batch": 4, "lmin": 262144, "lmax": 1048576, "nodes": 7, "heads": 16,
         "kv_heads": 4, "dim": 64, "block": 64, "window": 0, "first": 0, "sink": False, "softcap": 0.0, "spread": 3},
        # large trees in a sliding-window layer of wide heads that keeps its first four tokens, sink and softcap
        {"name": "tree_window", "kind": "tree", "batch": 6, "lmin": 100, "lmax": 8192, "nodes": 99, "heads": 16,
         "kv_heads": 1, "dim": 512, "block": 16, "window": 128, "first": 4, "sink": True, "softcap": 30.0, "spread": 4},
        # one chat's next token in a window of 128 behind four first tokens
        {"name": "stream_one", "kind": "stream", "batch": 1, "lmin": 5001, "lmax": 5001, "t_new": 1, "heads": 16,
         "kv_heads": 2, "dim": 128, "block": 16, "window": 128, "first": 4, "sink": False, "softcap": 0.0, "spread": 5},
        # a serving batch's next tokens in windows of 4k, some of the contexts shorter
        {"name": "stream_step", "kind": "stream", "batch": 64, "lmin": 2048, "lmax": 32768, "t_new": 1, "heads": 64,
         "kv_heads": 8, "dim": 128, "block": 64, "window": 4096, "first": 4, "sink": False, "softcap": 0.0, "spread": 6},
        # a prompt's chunk through windows of 2k behind 64 first tokens
        {"name": "stream_chunk", "kind": "stream", "batch": 2, "lmin": 16001, "lmax": 16384, "t_new": 1000, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 64, "window": 2048, "first": 64, "sink": True, "softcap": 0.0, "spread": 7},
        # the sampled token of one chat, with the five alternatives that an interface shows
        {"name": "score_one", "kind": "score", "rows": 1, "vocab": 32000, "type": "fp32", "top": 5, "masked": False},
        # a batch of small trees' nodes over a large vocabulary
        {"name": "score_step", "kind": "score", "rows": 256, "vocab": 131072, "type": "bf16", "top": 20, "masked": False},
        # a prompt's tokens over an odd vocabulary part of which a grammar forbids
        {"name": "score_prompt", "kind": "score", "rows": 3001, "vocab": 100003, "type": "fp16", "top": 8, "masked": True},
        # eight checked tokens of one chat
        {"name": "keep_one", "kind": "keep", "batch": 1, "lmin": 341, "lmax": 341, "nodes": 8, "kv_heads": 2, "dim": 128,
         "block": 16, "pools": 1, "spread": 24},
        # a serving batch's trees of up to 64 nodes in a cache of eight layers
        {"name": "keep_step", "kind": "keep", "batch": 64, "lmin": 1024, "lmax": 8192, "nodes": 64, "kv_heads": 8,
         "dim": 128, "block": 16, "pools": 8, "spread": 12},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the listed ranges."""
    while True:
        kind = rng.choice(["tree", "tree", "stream", "stream", "score", "score", "keep"])
        block = rng.choice([16, 32, 64, 64, 128])
        dim = rng.choice([32, 64, 64, 96, 128, 128, 160, 256, 512])
        if kind == "score":
            c = {"kind": kind, "rows": _log(rng, 1, 4096), "vocab": _log(rng, 1000, 200000),
                 "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "top": rng.choice([0, 1, rng.randint(2, 20), 64]),
                 "masked": rng.random() < 0.3}
            fits = c["rows"] * c["vocab"] <= 3001 * 100003
        elif kind == "keep":
            nodes = _log(rng, 2, 128)
            low = _log(rng, nodes, 4096)
            c = {"kind": kind, "batch": _log(rng, 1, 64), "lmin": low, "lmax": _log(rng, low, 8192), "nodes": nodes,
                 "kv_heads": rng.choice([1, 2, 3, 8]), "dim": dim, "block": block, "pools": rng.randint(1, 8),
                 "spread": rng.randrange(1 << 30)}
            fits = _pages(c) * block * c["kv_heads"] * dim * c["pools"] <= 2 ** 31
        else:
            kv = rng.choice([1, 1, 2, 4, 8])
            c = {"kind": kind, "batch": _log(rng, 1, 64)}
            if kind == "tree":
                t = c["nodes"] = _log(rng, 2, 128)
                window = rng.choice([0, 0, _log(rng, 1, 4096)])
            else:
                t = c["t_new"] = rng.choice([1, 1, _log(rng, 2, 1000)])
                window = _log(rng, 1, 4096)
            top = _log(rng, max(8, t), 524288 if t < 9 else 16384)
            c.update(lmin=max(t, int(top * rng.uniform(0.05, 1.0))), lmax=top, heads=kv * rng.choice([1, 3, 4, 8, 16]),
                     kv_heads=kv, dim=dim, block=block, window=window, first=_log(rng, 1, 200) if window else 0,
                     sink=rng.random() < 0.3, softcap=rng.choice([0.0, 0.0, 0.0, 30.0]), spread=rng.randrange(1 << 30))
            padded = c["batch"] * top
            fits = (padded * kv * dim <= 2 ** 31 and padded * c["heads"] * t <= 2 ** 30
                    and padded * c["heads"] * t * dim <= 2 ** 37)
        if fits:
            return c


def _lens(c: dict) -> list[int]:
    """The sequences' lengths, spread over the logarithm."""
    r = random.Random(c["spread"])
    return [_log(r, c["lmin"], c["lmax"]) for _ in range(c["batch"])]


def _new(c: dict) -> list[int]:
    """Nodes of each sequence's tree: of a larger batch fewer than the most in some, in one none."""
    if "nodes" not in c:
        return [c["t_new"]] * c["batch"]
    r = random.Random(c["spread"] + 1)
    got = [c["nodes"] if r.random() < 0.6 else r.randint(1, c["nodes"]) for _ in range(c["batch"])]
    if len(got) > 4:
        got[r.randrange(len(got))] = 0
    return got


def _trees(c: dict, forest: bool) -> list[list[int]]:
    """Each sequence's tree as its nodes' parents (-1: none); node 0 is a root, in a forest a few others too."""
    r = random.Random(c["spread"] + 2)
    trees = []
    for n in _new(c):
        wide = r.choice([2, 4, 8])  # a node hangs below one of so many before it, or below any
        tree = [-1]
        for t in range(1, n):
            near = r.randint(max(0, t - wide), t - 1) if r.random() < 0.7 else r.randrange(t)
            tree.append(-1 if forest and r.random() < 0.05 else near)
        trees.append(tree[:n])
    return trees


def _ancestors(tree: list[int], t: int) -> list[int]:
    got = []
    while t >= 0:
        got.append(t)
        t = tree[t]
    return got[::-1]


def _pages(c: dict) -> int:
    return sum(-(-n // c["block"]) for n in _lens(c))


def _row_bytes(c: dict) -> int:
    return c["kv_heads"] * c["dim"] * 17 // 16  # K and V of a token: codes and scales


def _histories(c: dict) -> list[list[int]]:
    """Each sequence's tokens' histories, as their lengths."""
    lens, new = _lens(c), _new(c)
    if c["kind"] == "stream":
        return [[n - m + t + 1 for t in range(m)] for n, m in zip(lens, new)]
    return [[n - m + len(_ancestors(tree, t)) for t in range(m)] for n, m, tree in zip(lens, new, _trees(c, True))]


def work(c: dict) -> dict:
    if c["kind"] == "score":
        size = 4 if c["type"] == "fp32" else 2
        return {"bytes": c["rows"] * (c["vocab"] * size + 12 + 8 * c["top"]), "flops": 0}
    if c["kind"] == "keep":
        moved = sum(1 for path in _paths(c) for i, p in enumerate(path) if p != i)
        nodes = sum(_new(c))
        # rows read and written; parents, tokens, picks read, masks, depths and paths written
        return {"bytes": 2 * moved * _row_bytes(c) * c["pools"] + nodes * (12 + 8 * -(-c["nodes"] // 64) + 8), "flops": 0}
    rows, pairs = 0, 0
    for n, m, hist in zip(_lens(c), _new(c), _histories(c)):
        seen = [min(h, c["first"] + c["window"]) if c["window"] else h for h in hist]
        pairs += sum(seen)
        rows += min(n, c["first"] + c["window"] + m - 1) if c["window"] and m else n if m else 0
    q = c["heads"] * c["dim"] * sum(_new(c))
    out = c["heads"] * c["dim"] * c["batch"] * c.get("nodes", c.get("t_new"))
    masks = 8 * -(-c["nodes"] // 64) * sum(_new(c)) if c["kind"] == "tree" else 0
    return {"bytes": rows * _row_bytes(c) + 2 * q + 2 * out + masks, "flops": 4 * pairs * c["heads"] * c["dim"]}


def _paths(c: dict) -> list[list[int]]:
    """The nodes that the model accepts: from the root towards one of the deeper nodes, as far as none of their rows is
    both moved and moved onto (so that a pass leaves the rows that the next one moves)."""
    r = random.Random(c["spread"] + 3)
    got = []
    for tree in _trees(c, False):
        path = max((_ancestors(tree, r.randrange(len(tree))) for _ in range(3)), key=len) if tree else []
        while not all(p == i or p >= len(path) for i, p in enumerate(path)):
            path.pop()
        got.append(path)
    return got


# ---------------------------------------------------------------------------
# The 4-bit format in elementary operations
# ---------------------------------------------------------------------------
def _pow2(e: torch.Tensor) -> torch.Tensor:
    return ((e.int() + 127) << 23).view(F32)


def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (packed two a byte) and scale bytes of x [..., D]: per 32 dims the smallest power of two under which no
    value passes 6, each value rounded to the nearest level."""
    b = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(m > 0.75, e - 2, e - 3).clamp(-120, 125)
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


def _tables(c: dict, seed: int, lens: list[int], n_pages: int) -> tuple[torch.Tensor, list[int]]:
    """A block table over a random permutation of the pages, and the ids that are left, in the order of their use."""
    order = list(range(n_pages))
    random.Random(seed).shuffle(order)
    width = max(1, max(-(-n // c["block"]) for n in lens))
    bt = torch.full((len(lens), width), -1, dtype=I32)
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
    if c["kind"] == "score":
        return _prepare_score(c, gen, s)
    lens, new = _lens(c), _new(c)
    if c["kind"] == "keep":
        return _prepare_keep(c, seed, gen, s, lens, new)
    n_pages = _pages(c) + 3
    s["pool"] = _pool(c, n_pages)
    s["bt"], _ = _tables(c, seed, lens, n_pages)
    s["lens"] = torch.tensor(lens, dtype=I32, device=dev)
    _fill(c, s["pool"], gen)
    t = c.get("nodes", c.get("t_new"))
    s["q"] = torch.randn(c["batch"], t, c["heads"], c["dim"], generator=gen, device=dev).to(BF)
    s["sink"] = torch.randn(c["heads"], generator=gen, device=dev) if c["sink"] else None
    s["max_len"] = max(lens)
    s["n_new"], s["tree"] = None, None
    if c["kind"] == "tree":
        s["n_new"] = torch.tensor(new, dtype=I32, device=dev)
        # the step's masks, which every layer's attention takes: bit j of node t's words: it sees node j
        masks = torch.zeros(c["batch"], t, -(-t // 64) * 64, dtype=I64)
        for b, tree in enumerate(_trees(c, True)):
            for i in range(len(tree)):
                masks[b, i, _ancestors(tree, i)] = 1
        s["tree"] = (masks.unflatten(-1, (-1, 64)) << torch.arange(64)).sum(-1).to(dev)
    return s


def _prepare_score(c: dict, gen: torch.Generator, s: dict) -> dict:
    dev = _dev()
    shape = (c["rows"], c["vocab"])
    # rows from nearly even to peaked
    x = torch.randn(shape, generator=gen, device=dev) * (0.5 + 5 * torch.rand(c["rows"], 1, generator=gen, device=dev))
    if c["masked"]:  # half of the vocabulary, in a third of the rows
        part = torch.rand(c["rows"], 1, generator=gen, device=dev) < 0.34
        x = x.masked_fill(part & (torch.rand(shape, generator=gen, device=dev) < 0.5), -math.inf)
    s["logits"] = x.to(TYPES[c["type"]])
    tokens = torch.randint(0, c["vocab"], (c["rows"],), generator=gen, device=dev)
    likely = x.argmax(-1)
    pick = torch.rand(c["rows"], generator=gen, device=dev)
    tokens = torch.where(pick < 0.5, likely, tokens)
    if c["rows"] > 8:  # rows of padding, that ask for no token
        tokens = torch.where(pick > 0.97, torch.full_like(tokens, -1), tokens)
    s["tokens"] = tokens
    return s


def _prepare_keep(c: dict, seed: int, gen: torch.Generator, s: dict, lens: list[int], new: list[int]) -> dict:
    dev = _dev()
    n_pages = _pages(c) + 3
    bt, free = _tables(c, seed, lens, n_pages)
    # tables, lengths and the free stack in one buffer: a pass starts from the kept copy of it
    parts = [bt.flatten(), torch.tensor(lens, dtype=I32, device=dev),
             torch.tensor(free[::-1] + [0] * (n_pages - len(free)), dtype=I32, device=dev),
             torch.tensor([len(free)], dtype=I32, device=dev), torch.zeros(1, dtype=I32, device=dev)]
    sizes = [-(-p.numel() // 4) * 4 for p in parts]
    s["kept"] = torch.cat([torch.nn.functional.pad(p, (0, n - p.numel())) for p, n in zip(parts, sizes)])
    s["books"] = s["kept"].clone()
    views = s["books"].split(sizes)
    s["bt"] = views[0][:bt.numel()].view(bt.shape)
    for name, v, p in zip(("lens", "stack", "top", "status"), views[1:], parts[1:]):
        s[name] = v[:p.numel()]
    r = random.Random(seed)
    parents, tokens, picks = (torch.full((c["batch"], c["nodes"]), -1, dtype=I32) for _ in range(3))
    for b, (tree, path) in enumerate(zip(_trees(c, False), _paths(c))):
        # drafts of siblings differ; off the path the model picks what was not drafted
        names = r.sample(range(100000), 2 * len(tree) + 1)
        token, pick = names[:len(tree)], names[len(tree):2 * len(tree)]
        for p, q in zip(path, path[1:]):
            pick[p] = token[q]
        if tree:
            parents[b, :len(tree)], tokens[b, :len(tree)], picks[b, :len(tree)] = map(torch.tensor, (tree, token, pick))
    s["parents"], s["tokens"], s["picks"] = parents.to(dev), tokens.to(dev), picks.to(dev)
    s["n_new"] = torch.tensor(new, dtype=I32, device=dev)
    s["refs"] = torch.zeros(n_pages, dtype=I32, device=dev)
    s["pools"] = []
    for _ in range(c["pools"]):
        pool = _pool(c, n_pages)
        pool.view(-1).view(I64).random_(generator=gen)  # a page is whole blocks of 16 tokens
        s["pools"].append(pool)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s: dict):
    c = s["case"]
    if own:
        kv = _api()
        if c["kind"] == "score":
            return tuple(kv.ops.token_logprobs(s["logits"], s["tokens"], top=c["top"]))
        if c["kind"] != "keep":
            return kv.fp4_attention(s["q"], s["pool"], s["bt"], s["lens"], n_new=s["n_new"], window=c["window"] or None,
                                    first=c["first"], tree=s["tree"], sink=s["sink"], softcap=c["softcap"] or None,
                                    max_len=s["max_len"])
        s["books"].copy_(s["kept"])
        tree, depths = kv.ops.draft_tree(s["parents"], s["n_new"])
        path, n_keep, following = kv.ops.accept_drafts(s["parents"], s["tokens"], s["picks"], s["n_new"])
        kv.ops.keep_tokens(s["stack"], s["top"], s["bt"], s["lens"], s["n_new"], path, n_keep, s["pools"], s["status"],
                           refs=s["refs"])
        return [tree, depths, path, n_keep, following, s["books"], *s["pools"]]
    if c["kind"] == "score":
        return _plain_score(s)
    if c["kind"] != "keep":
        return _plain_attend(s)
    s["books"].copy_(s["kept"])
    seen = _plain_tree(s)
    path, n_keep, following = _plain_accept(s, seen)
    _plain_keep(s, path, n_keep)
    words = torch.nn.functional.pad(seen.long(), (0, -seen.shape[2] % 64)).unflatten(-1, (-1, 64))
    tree = (words << torch.arange(64, device=words.device)).sum(-1)
    depths = (seen.sum(-1) - 1).clamp_min(0).to(I32)
    return [tree, depths, path, n_keep, following, s["books"], *s["pools"]]


def _plain_score(s: dict):
    """Log probability of each row's token (0 where it is negative), entropy, and the most likely tokens (ties: the
    lowest) with their log probabilities."""
    c = s["case"]
    x = s["logits"].float() + 0.0
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(-1)
    norm = torch.log(total)
    entropy = norm - (e * d.masked_fill(e == 0, 0.0)).sum(-1) / total
    got = d.gather(1, s["tokens"].clamp_min(0)[:, None])[:, 0] - norm
    got = torch.where(s["tokens"] < 0, torch.zeros_like(got), got)
    bits = x.view(I32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    order = (order << 32) + torch.arange(c["vocab"] - 1, -1, -1, device=x.device)
    ids = c["vocab"] - 1 - (torch.topk(order, c["top"], dim=-1).values & 0xFFFFFFFF)
    return got, entropy, ids.to(I32), d.gather(1, ids) - norm[:, None]


def _plain_attend(s: dict) -> torch.Tensor:
    c = s["case"]
    kv, g, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    t = s["q"].shape[1]
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
    # which of a sequence's positions a token sees: those before the new ones, and of these the ones of its mask
    step = torch.arange(t, device=a.device)
    if s["tree"] is None:
        mask = (step[:, None] >= step).expand(c["batch"], t, t)
        base = s["lens"].long() - t
    else:
        mask = (s["tree"].unsqueeze(-1) >> torch.arange(64, device=a.device) & 1).flatten(2)[..., :t] > 0
        base = (s["lens"] - s["n_new"]).long()
    pos = torch.arange(n, device=a.device)
    at = (pos - base[:, None]).clamp(0, t - 1)  # [B, n]
    new = mask.gather(2, at[:, None].expand(-1, t, -1)) & (pos < s["lens"][:, None])[:, None]
    old = (pos < base[:, None])[:, None]
    seen = torch.where(old, mask.any(-1, keepdim=True), new)
    if c["window"]:
        place = mask.long().cumsum(-1) - 1 + base[:, None, None]  # of the masked tokens in the history
        place = torch.where(old, pos, place.gather(2, at[:, None].expand(-1, t, -1)))
        whole = base[:, None, None] + mask.sum(-1, keepdim=True)
        seen = seen & ((place < c["first"]) | (place >= whole - c["window"]))
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


def _plain_tree(s: dict) -> torch.Tensor:
    """[B, T, T]: node t's ancestors and itself, by products that double the steps upwards."""
    t = s["parents"].shape[1]
    step = torch.arange(t, device=s["parents"].device)
    live = step < s["n_new"][:, None]
    up = ((s["parents"][..., None] == step) | (step[:, None] == step)) & live[..., None]
    reach = up.float()
    for _ in range(max(1, (t - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach > 0


def _plain_accept(s: dict, seen: torch.Tensor):
    """From the root on, the child whose token is the one that the model picked after its parent (the first of equal
    ones): the path, its length and what is picked after it."""
    parents = s["parents"].long()
    t = parents.shape[1]
    step = torch.arange(t, device=parents.device)
    wanted = (parents >= 0) & (step < s["n_new"][:, None]) & (s["tokens"] == s["picks"].gather(1, parents.clamp_min(0)))
    twin = wanted[:, None, :] & (parents[:, None, :] == parents[..., None]) & (step < step[:, None])
    good = (wanted & ~twin.any(-1)) | (step == 0)
    on = (seen <= good[:, None, :]).all(-1) & seen[..., 0]
    n_keep = on.sum(-1)
    place = torch.where(on, on.long().cumsum(-1) - 1, torch.full_like(parents, t))
    path = torch.full((parents.shape[0], t + 1), -1, dtype=I32, device=parents.device)
    path.scatter_(1, place, step.to(I32).expand_as(place))
    path = path[:, :t]
    end = path.gather(1, (n_keep - 1).clamp_min(0)[:, None]).clamp_min(0).long()
    following = torch.where(n_keep > 0, s["picks"].gather(1, end)[:, 0], torch.full_like(s["picks"][:, 0], -1))
    return path, n_keep.to(I32), following


def _plain_keep(s: dict, path: torch.Tensor, n_keep: torch.Tensor) -> None:
    """Token path[i] of the new ones becomes token i; the length ends behind the last of them; pages behind it go on the
    free stack: sequences ascending, a sequence's pages from its last to its first."""
    c, bt, lens = s["case"], s["bt"], s["lens"]
    base = (lens - s["n_new"]).long()
    b, i = (path >= 0).nonzero(as_tuple=True)
    src, dst = base[b] + path[b, i], base[b] + i
    from_page, from_slot = bt[b, src // c["block"]].long(), src % c["block"]
    to_page, to_slot = bt[b, dst // c["block"]].long(), dst % c["block"]
    for pool in s["pools"]:
        for plane in _planes(pool, c["block"], c["dim"]):
            plane[to_page, :, to_slot] = plane[from_page, :, from_slot]
    held = (lens + c["block"] - 1) // c["block"]
    lens.copy_((base + n_keep).to(I32))
    left = (lens + c["block"] - 1) // c["block"]
    at = torch.arange(bt.shape[1], device=bt.device)[None]
    gone = (at >= left[:, None]) & (at < held[:, None])
    push = bt.flip(1)[gone.flip(1)]
    s["stack"][s["top"].long() + torch.arange(push.shape[0], device=bt.device)] = push
    s["top"].add_(push.shape[0])
    bt.masked_fill_(gone, -1)


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
    if c["kind"] == "keep":
        return None
    s = prepare(c, seed)
    if c["kind"] == "score":
        got, entropy = (torch.zeros(c["rows"], dtype=F64, device=_dev()) for _ in range(2))
        likely = torch.zeros(c["rows"], c["top"], dtype=F64, device=_dev())
        step = max(1, 2 ** 26 // c["vocab"])
        for r in range(0, c["rows"], step):
            p = torch.log_softmax(s["logits"][r:r + step].double(), -1)
            tok = s["tokens"][r:r + step]
            got[r:r + step] = torch.where(tok < 0, 0.0, p[torch.arange(p.shape[0], device=p.device), tok])
            entropy[r:r + step] = torch.special.entr(p.exp()).sum(-1)
            likely[r:r + step] = p.sort(-1, descending=True).values[:, :c["top"]]
        return got, entropy, None, likely
    lens, new = _lens(c), _new(c)
    if 4.0 * sum(n * m for n, m in zip(lens, new)) * c["heads"] * c["dim"] > 3e13:
        return None
    trees = _trees(c, True) if c["kind"] == "tree" else [list(range(-1, n - 1)) for n in new]
    g = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=F64, device=s["q"].device)
    for b, (n, m, tree) in enumerate(zip(lens, new, trees)):
        if m == 0:
            continue
        hidden = torch.ones(m, n, dtype=torch.bool)
        for t in range(m):
            history = list(range(n - m)) + [n - m + j for j in (_ancestors(tree, t) if s["tree"] is not None else range(t + 1))]
            if c["window"]:
                history = history[:c["first"]] + history[max(c["first"], len(history) - c["window"]):]
            hidden[t, torch.tensor(history)] = False
        hidden = hidden.to(out.device)
        pages = s["bt"][b, :-(-n // c["block"])]
        for h in range(c["kv_heads"]):
            k, v = _exact_rows(s["pool"], pages, h, n, c["block"], c["dim"])
            for i in range(h * g, (h + 1) * g):
                a = s["q"][b, :m, i].double() @ k.T / math.sqrt(c["dim"])
                if c["softcap"]:
                    a = c["softcap"] * torch.tanh(a / c["softcap"])
                a = a.masked_fill(hidden, -math.inf)
                if s["sink"] is not None:
                    a = torch.cat([a, s["sink"][i].double().expand(m, 1)], 1)
                out[b, :m, i] = torch.softmax(a, 1)[:, :n] @ v
    return out
