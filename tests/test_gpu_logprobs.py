"""Log probabilities, entropy and the most likely tokens against numpy in 64 bits.

Ids are equal.  Tolerances, with u = 2^-24 (half a step of fp32), d = x - m:
* l = sum exp(d): d and d log2(e) are rounded (2 u |d| together), the exponential is off by 2 u, so a term by
  u e^d (2 |d| + 2) <= 3 u of l's scale (e^d |d| <= 0.37, and l >= 1).  A running sum is rescaled at most once for every
  chunk of its lane, wave and segment, each time off by 5 u of itself, and added to as often; within a chunk, across
  lanes, waves and segments some 24 sums follow each other.  With up to 40 chunks: 3 + 40 * 6 + 24 + rescalings of the
  joins, below 300 u of l.  ln l is off by that and 3 u |ln l| of the logarithm.
* logprob = (x - m) - ln l: 300 u + 3 u |ln l| + u |x - m| + u |logprob|.
* entropy = ln l - s / l: s is off as l is, a term's weight by u (2 |d| + 2) and its d by u |d|: together
  300 u (|s / l| + 1) + 4 u sum p d^2 + 4 u (|ln l| + |s / l|).
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle.token_logprobs import token_logprobs as oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def check(got, x: torch.Tensor, tokens: torch.Tensor | None, top: int, times: int = 1) -> None:
    """Of rows that each came ``times`` times, one after another."""
    x = x.float().cpu().double().numpy().reshape(-1, x.shape[-1])
    t = np.full(x.shape[0], -1) if tokens is None else tokens.cpu().numpy().reshape(-1)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        lp, h, ids, best = oracle(x, t, top)
        m = x.max(-1)
        d = x - m[:, None]
        e = np.where(np.isfinite(d), np.exp(d), 0.0)
        total = e.sum(-1)
        norm = np.log(total)
        dz = np.where(e > 0, d, 0.0)
        mean, square = (e * dz).sum(-1) / total, (e * dz * dz).sum(-1) / total
    lp, h, ids, best, norm, mean, square = (np.repeat(a, times, 0) for a in (lp, h, ids, best, norm, mean, square))
    assert np.array_equal(got.top_ids.cpu().numpy().reshape(ids.shape), ids)

    def near(g, want, bound):
        g = g.cpu().double().numpy().reshape(want.shape)
        # past fp32's range (a logit of -3e38 below one of 3e38: -6e38 > 2^128) the rounded value is an infinity
        want = np.where(np.abs(want) >= 2.0 ** 128, np.sign(want) * np.inf, want)
        assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(g[np.isinf(want)], want[np.isinf(want)])
        fine = np.isfinite(want)
        off = np.abs(g[fine] - want[fine]) - np.broadcast_to(bound, want.shape)[fine]
        assert (off <= 0).all(), f"worst {off.max()} of {np.abs(want[fine]).max()}"

    base = 300 * U + 3 * U * np.abs(norm)

    def of(p):
        with np.errstate(invalid="ignore"):
            return U * np.abs(p) + U * np.abs(p + norm.reshape(-1, *[1] * (p.ndim - 1)))

    if tokens is None:
        assert got.logprobs is None
    else:
        near(got.logprobs, lp, base + of(lp))
    near(got.entropy, h, 300 * U * (np.abs(mean) + 1) + 4 * U * square + 4 * U * (np.abs(norm) + np.abs(mean)))
    near(got.top_logprobs, best, base[:, None] + of(best))


def inputs(dev, rows, vocab, kind, seed, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device=dev) * scale).to(TYPES[kind])
    t = torch.randint(-1, vocab, (rows,), generator=g, device=dev)
    return x, t


# one vector and less, a wave's and a workgroup's chunk and the sizes about them, odd ones, several segments
SIZES = [1, 2, 7, 8, 9, 63, 64, 100, 513, 1000, 2047, 2049, 4096, 8191, 8193, 16384, 32000, 50257, 100003, 262145, 300007]


@pytest.mark.parametrize("vocab", SIZES)
@pytest.mark.parametrize("kind", TYPES)
def test_sizes(dev, vocab, kind) -> None:
    from saint_kv import ops

    for rows, top in ((1, 5), (3, 64), (2, 0), (5, 1)):
        top = min(top, vocab)
        x, t = inputs(dev, rows, vocab, kind, seed=vocab + rows)
        check(ops.token_logprobs(x, t, top=top), x, t, top)
    check(ops.token_logprobs(x), x, None, 0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1500, 1000, 20), (1100, 5003, 3), (2100, 300, 64), (400, 20011, 20)])
def test_many_rows(dev, rows, vocab, top, kind) -> None:
    """A workgroup a row, or a few."""
    from saint_kv import ops

    x, t = inputs(dev, rows, vocab, kind, seed=rows)
    got = ops.token_logprobs(x, t.to(torch.int32), top=top)
    check(got, x, t, top)
    again = ops.token_logprobs(x, t, top=top)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def special_rows(vocab: int) -> torch.Tensor:
    """Rows that break a running maximum, a bound or a sum."""
    g = torch.Generator().manual_seed(1)
    r = torch.randn(vocab, generator=g)
    inf, low = math.inf, torch.finfo(torch.float32).min
    i = torch.arange(vocab)
    rows = [torch.zeros(vocab), torch.full((vocab,), -inf), torch.full((vocab,), low), r.sort().values, r.sort(descending=True).values,
            torch.where(i == vocab // 2, r, torch.tensor(-inf)), torch.where(i % 3 == 0, r, torch.tensor(-inf)),
            torch.where(i < 5, r, torch.tensor(low)), torch.where(i == 7, torch.tensor(inf), r),
            torch.where((i == 3) | (i == vocab - 1), torch.tensor(math.nan), r), torch.where(i % 2 == 0, 0.0, -0.0),
            (r > 0).float(), (r * 2).round(), torch.where(i // 8 % 256 < 3, r + 9, r), torch.where(i // 4 % 256 < 2, 9.0, r),
            r * 1e-3 + 80, r * 30, torch.where(i == 1, 3e38, -3e38), torch.where(i == vocab - 1, 60.0, r),
            torch.where(i == 0, torch.tensor(-math.nan), r)]
    return torch.stack(rows)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab", [70, 3001, 20000, 70001])
def test_special_rows(dev, kind, vocab) -> None:
    """Equal logits throughout, nothing but -inf or the lowest value, NaN and infinities, ties of zeros, the best in few lanes."""
    from saint_kv import ops

    x = special_rows(vocab)
    if kind == "bf16":
        x = x.clamp_min(torch.finfo(torch.bfloat16).min).where(x != -math.inf, x)  # the lowest value stays finite
    if kind == "fp16":
        x = x.clamp(-60000, 60000).where(torch.isfinite(x), x)
    x = x.to(TYPES[kind]).to(dev)
    t = torch.arange(x.shape[0], device=dev) % vocab
    for top in (0, 1, 20, 64):
        check(ops.token_logprobs(x, t, top=top), x, t, top)
        many = x.repeat_interleave(60, 0)  # a workgroup a row
        check(ops.token_logprobs(many, t.repeat_interleave(60), top=top), x, t, top, times=60)


@pytest.mark.parametrize("kind", TYPES)
def test_strides_and_shapes(dev, kind) -> None:
    """Rows that begin anywhere, a wider buffer's columns, more dims, ids of other strides, rows behind left out."""
    from saint_kv import ops

    x, _ = inputs(dev, 6, 5003, kind, seed=1)
    for view in (x[:, 1:], x[:, 3:4100], x[::2, 5:], x[1:].unflatten(0, (5, 1)), x.unflatten(0, (2, 3))[:, :2, 7:], x[2],
                 x[:1].expand(4, -1), x[:0]):
        lead = view.shape[:-1]
        if view.dim() == 3 and lead[1] == 2:  # rows of two strides
            with pytest.raises(ValueError, match="stride"):
                ops.token_logprobs(view, top=4)
            continue
        ids = torch.randint(0, view.shape[-1], (*lead, 2), device=dev)[..., 0]
        got = ops.token_logprobs(view, ids, top=4)
        assert got.logprobs.shape == lead and got.top_ids.shape == (*lead, 4)
        if view.numel():
            check(got, view.contiguous(), ids, 4)


def test_tokens_outside_the_vocabulary(dev) -> None:
    from saint_kv import ops

    x, _ = inputs(dev, 4, 100, "fp32", seed=1)
    got = ops.token_logprobs(x, torch.tensor([-1, 100, 1 << 40, -(1 << 40)], device=dev)).logprobs
    assert got[0] == 0 and torch.isnan(got[1:3]).all() and got[3] == 0


def test_refusals(dev) -> None:
    from saint_kv import ops

    x, t = inputs(dev, 2, 400000, "bf16", seed=1)  # in segments, so with a workspace
    for bad in (dict(logits=x.double()), dict(logits=x.t()), dict(logits=x[:, :0], tokens=None), dict(tokens=t[:1]),
                dict(tokens=t.float()), dict(top=-1), dict(top=65), dict(logits=x[:, :3], top=4),
                dict(workspace=torch.zeros(8, device=dev), top=4)):
        with pytest.raises(ValueError):
            ops.token_logprobs(**{**dict(logits=x, tokens=t), **bad})
    with pytest.raises(RuntimeError, match="CPU"):
        ops.token_logprobs(x.cpu())
    need = ops.token_logprobs_workspace(x, 4)
    assert need > 0
    got = ops.token_logprobs(x, t, top=4, workspace=torch.empty(need, dtype=torch.uint8, device=dev))
    check(got, x, t, 4)


def test_captured_calls_replay(dev) -> None:
    """Two graphs of their own workspaces, replayed in turn; the picks of one go on to accept drafts."""
    from saint_kv import ops

    x, t = inputs(dev, 12, 32000, "bf16", seed=1)
    y, _ = inputs(dev, 2000, 500, "fp32", seed=2)
    parents = torch.arange(-1, 5, dtype=torch.int32, device=dev).repeat(2, 1)
    tokens = torch.zeros(2, 6, dtype=torch.int32, device=dev)

    def step():
        got = ops.token_logprobs(x, t, top=3)
        return [*got, *ops.accept_drafts(parents, tokens, got.top_ids[:, 0].view(2, 6))]

    def other():
        return list(ops.token_logprobs(y, top=7)[1:])

    step(), other()
    torch.cuda.synchronize()
    graphs = []
    for f in (step, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, f, out))
    for n in range(4):
        x.copy_(inputs(dev, 12, 32000, "bf16", seed=10 + n)[0])
        y.copy_(inputs(dev, 2000, 500, "fp32", seed=20 + n)[0])
        tokens[:, 1:] = x.argmax(-1).view(2, 6)[:, :-1]
        tokens[1, 3] = -5
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, f, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, f()))
        assert graphs[0][2][-2].tolist() == [6, 3]


def test_calls_on_two_streams_at_once(dev) -> None:
    from saint_kv import ops

    cases = [(inputs(dev, 3, 300007, "bf16", seed=1), 20), (inputs(dev, 200, 32000, "fp32", seed=2), 64), (inputs(dev, 1500, 3000, "fp16", seed=3), 5)]
    want = [ops.token_logprobs(x, t, top=top) for (x, t), top in cases]
    streams = [torch.cuda.Stream(device=dev) for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream, ((x, t), top) in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(ops.token_logprobs(x, t, top=top))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 3]))


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_huge_logits_among_others(dev, kind) -> None:
    """Logits past 1e37 in a wave, a segment or a row of their own, above, below and beside ordinary ones."""
    from saint_kv import ops

    for vocab in (3000, 70001, 300007):
        x, t = inputs(dev, 8, vocab, kind, seed=vocab)
        x[0, 17] = 2e38
        x[1, ::3] = -2e38
        x[2, : vocab // 2] = -3e38
        x[3] = 1e38
        x[4] = -1e38
        x[4, vocab - 1] = -0.99e38
        x[5, 1:] = -3e38
        x[6, vocab // 2:] = 3e38
        x[7] = x[7].abs() * 1e37
        check(ops.token_logprobs(x, t, top=6), x, t, 6)


@pytest.mark.parametrize("scale", [1e5, 1e7, 6e7, 1e8, 1e9, 1e12, 1e20, 1e30, 1e36])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_logits_of_any_size(dev, kind, scale) -> None:
    """All of a row's logits large, of both signs, of one, close together, and some lanes' alone."""
    from saint_kv import ops

    for rows, vocab in ((5, 32000), (700, 3001)):
        x, t = inputs(dev, rows, vocab, "fp32", seed=rows)
        x = x * scale
        x[1].abs_()
        x[2] = -x[2].abs()
        x[3] = scale * (1 + 2.0 ** -20 * torch.arange(vocab, device=dev) / vocab)
        x[4, 300:] = 0.01
        x = x.to(TYPES[kind])
        check(ops.token_logprobs(x, t, top=5), x, t, 5)


@pytest.mark.parametrize("mask", [-1e4, -1e7, -1e9, -1e20, -1e30, -1e34, -1e35, -1e36, -5e36, -9.9e36, -1.1e37])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_masks_far_below_the_rest(dev, kind, mask) -> None:
    """Lanes and waves that see nothing but a finite mask, many times over: their sum times the way up to the maximum
    passes fp32, and counts for nothing."""
    from saint_kv import ops

    for rows, vocab in ((2, 32000), (1, 262145), (700, 32000), (700, 3001)):
        x, t = inputs(dev, rows, vocab, kind, seed=rows)
        x[:, 9:vocab - 1] = mask
        x[0] = mask
        x[-1, :40] = mask
        check(ops.token_logprobs(x, t, top=5), x, t, 5)


@pytest.mark.parametrize("rows,vocab", [(5, 5001), (3, 200003), (1100, 700)])
def test_far_rows(dev, rows, vocab) -> None:
    """Rows whose bytes lie past 2^32."""
    from saint_kv import ops

    stride = (3 << 30) // rows // 8 * 8 + 3
    buffer = torch.empty(stride * rows, dtype=torch.bfloat16, device=dev)
    assert stride * (rows - 1) * 2 > 2 ** 32
    far = buffer.view(rows, stride)[:, :vocab]
    x, t = inputs(dev, rows, vocab, "bf16", seed=vocab)
    far.copy_(x)
    got = ops.token_logprobs(far, t, top=7)
    check(got, x, t, 7)


@pytest.mark.parametrize("lead", [(0,), (5, 0), (0, 5), (3, 0, 2), (1, 0)])
def test_no_rows(dev, lead) -> None:
    """A dimension of no rows anywhere: outputs of as many."""
    from saint_kv import ops

    x = torch.zeros(*lead, 50, dtype=torch.bfloat16, device=dev)
    got = ops.token_logprobs(x, torch.zeros(lead, dtype=torch.int64, device=dev), top=4)
    assert got.logprobs.shape == got.entropy.shape == lead and got.top_ids.shape == got.top_logprobs.shape == (*lead, 4)
    assert ops.token_logprobs_workspace(x, 4) == 0
