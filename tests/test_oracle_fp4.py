"""The oracle of the 4-bit token cache against hand-worked codes and the nearest value."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import fp4_cache as ora


def test_levels() -> None:
    assert ora.LEVELS.tolist() == [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def test_codes_by_hand() -> None:
    x = np.zeros(32)
    x[:16] = [6, -6, 5, 5.01, 0.25, 0.26, -0.75, 1.25, 1.75, 2.5, 3.5, 2.49, -0.0, 4.99, 0.74, 3.51]
    codes, scale = ora.quantize(x)
    assert scale.tolist() == [127]  # 2^0: 6 fits
    assert codes[:16].tolist() == [7, 15, 6, 7, 0, 1, 10, 2, 4, 4, 6, 4, 8, 6, 1, 6]
    codes, scale = ora.quantize(np.where(np.arange(32) == 3, 6.001, x))
    assert scale.tolist() == [128]  # 6.001 does not
    assert ora.quantize(np.zeros(32))[1].tolist() == [7]
    assert ora.quantize(np.full(32, 3e38))[1].tolist() == [252]
    assert ora.dequantize(*ora.quantize(np.full(32, 3e38)))[0] == 6 * 2.0 ** 125


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_block_that_is_not_finite_reads_as_nan(bad: float) -> None:
    x = np.ones((2, 64))
    x[1, 40] = bad
    v = ora.dequantize(*ora.quantize(x))
    assert np.isnan(v[1, 32:]).all() and (v[0] == 1).all() and (v[1, :32] == 1).all()


def test_nearest_of_all_values() -> None:
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)) * 2.0 ** rng.integers(-30, 30, (200, 1))
    codes, scales = ora.quantize(x)
    step = np.repeat(2.0 ** (scales.astype(float) - 127), 32, -1)
    assert (np.abs(x) <= 6 * step).all()
    assert (np.abs(x).reshape(200, 2, 32).max(-1) > 3 * step[:, ::32]).all()  # half the scale is too small
    every = np.concatenate([ora.LEVELS, -ora.LEVELS])[:, None, None] * step
    assert np.array_equal(np.abs(every - x).min(0), np.abs(ora.dequantize(codes, scales) - x))


def test_pages_round_trip_and_layout() -> None:
    rng = np.random.default_rng(1)
    pool = np.zeros((3, 16, 2, 34 * 2), dtype=np.uint8)  # 2 heads of 64 dims
    k, v = rng.standard_normal((1, 20, 2, 64)), rng.standard_normal((1, 20, 2, 64))
    bt = np.array([[2, 0]], dtype=np.int32)
    ora.append(pool, bt, np.array([20]), k, v, np.array([20]))
    kk, vv, mapped = ora.rows(pool, bt, 0, range(20))
    assert mapped.all()
    assert np.array_equal(kk, ora.dequantize(*ora.quantize(k[0])))
    assert np.array_equal(vv, ora.dequantize(*ora.quantize(v[0])))
    # token 17, head 1: slot 1 of page 0; value scale bytes behind both code planes and its key's
    flat = pool.reshape(3, 2, -1)
    assert flat[0, 1, 2 * 16 * 32 + 1 * 4 + 2: 2 * 16 * 32 + 1 * 4 + 4].tolist() == \
        ora.quantize(v[0, 17, 1])[1].tolist()


def test_attention_of_equal_scores_is_the_mean() -> None:
    rng = np.random.default_rng(2)
    pool = np.zeros((2, 16, 1, 34), dtype=np.uint8)
    k, v = rng.standard_normal((1, 20, 1, 32)), rng.standard_normal((1, 20, 1, 32))
    bt = np.array([[1, 0]], dtype=np.int32)
    ora.append(pool, bt, np.array([20]), k, v, np.array([20]))
    _, vv, _ = ora.rows(pool, bt, 0, range(20))
    out = ora.attention(np.zeros((1, 2, 3, 32)), pool, bt, np.array([20]))
    assert np.allclose(out[0, 1], vv[:, 0].mean(0)) and np.allclose(out[0, 0], vv[:19, 0].mean(0))
    out = ora.attention(np.zeros((1, 1, 1, 32)), pool, bt, np.array([20]), window=4, sink=np.zeros(1))
    assert np.allclose(out[0, 0, 0], vv[16:, 0].sum(0) / 5)  # the sink is a fifth key without a value
    assert (ora.attention(np.ones((1, 3, 1, 32)), pool, bt, np.array([1]))[0, :2] == 0).all()
