"""Statistics of the layer norm where the mean is large against the deviations, against the definition in
extended precision on the stored inputs.

Tolerances, with u the rounding of the stat type and R = |mean| / deviation: a sum of a row goes through at
most 32 additions one after the other (a thread's share, the warp, the block) and a product, so the first
mean is off by at most P = 34 u R deviations.  Differences from it are exact, their sum is off by 34 u (0.8
+ P) deviations, and the variance by 36 u (1 + P^2) + 68 u P (0.8 + P) of itself: the inverse deviation by
less than 55 u (1 + P)^2 of itself, a result by less than 110 u (1 + P)^2 of the row's largest."""
import numpy as np
import pytest

import eshkol_b200 as eb
from eshkol_b200 import inputs
from test_gpu_norm_logprobs import done, kinds, laid, room, wide64

pytestmark = pytest.mark.gpu


def definition(xs, eps):
    """(y, mean, inv_std) in extended precision, of the differences from a row's first entry: these are exact
    for rows far from zero, where sums of the entries themselves would lose 2^-64 of the mean"""
    x = xs.astype(np.longdouble)
    first = x[:, :1]
    shift = (x - first).sum(axis=1, keepdims=True) / x.shape[1]
    d = (x - first) - shift
    inv = 1.0 / np.sqrt((d * d).sum(axis=1, keepdims=True) / x.shape[1] + np.longdouble(eps))
    return d * inv, (first + shift)[:, 0], inv[:, 0]


def forward(x, rows, n, tag, wt, eps):
    t = x.dtype
    y, mean, inv = room((rows, n), t), room((rows,), wt), room((rows,), wt)
    eb.layernorm_device(x.data_ptr(), 0, 0, y.data_ptr(), mean.data_ptr(), inv.data_ptr(), rows, n, eps, tag, ldx=x.stride(0))
    done()
    return wide64(y), wide64(mean), wide64(inv)


# a warp a row, a block a row (few and many rows), rows off the 16-byte boundaries, rows read three times
@pytest.mark.parametrize("rows,n,pad", [(700, 120, 0), (60, 2048, 0), (700, 4099, 0), (40, 1001, 1), (3, 20000, 0)])
@pytest.mark.parametrize("dtype,ratio", [("f32", 1e3), ("f32", 1e4), ("f32", 1e5), ("f32", 1e6), ("f64", 1e6), ("f64", 1e8),
                                         ("f64", 1e10)])
def test_mean_far_above_the_deviations(gpu_lib, dtype, ratio, rows, n, pad):
    t, tag, wt, u, half = kinds(dtype)
    x = laid(inputs.normal(131, (rows, n)) - ratio, t, pad)
    y, mean, inv = forward(x, rows, n, tag, wt, 0.0)
    want, wm, wi = definition(wide64(x), 0.0)
    grow = (1.0 + 34 * u * ratio * 1.2) ** 2  # a short row's deviation may be a little below one
    assert np.all(np.abs(inv - wi) <= 55 * u * grow * wi)
    assert np.all(np.abs(y - want) <= 110 * u * grow * np.abs(want).max(axis=1, keepdims=True))
    assert np.all(np.abs(mean - wm) <= 3 * u * np.abs(wm) + 40 * u * (1.0 + 34 * u * ratio))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(600, 96), (8, 4000), (700, 3900)])
def test_nearly_constant_rows_of_16_bits(gpu_lib, dtype, rows, n):
    """All entries but one are the same number and that one is a step below it: the variance is a small
    share of a step's square, and the pivot must not be a step away.  Sums of these numbers are exact up to
    the variance's own: 55 u of the inverse deviation."""
    import torch
    t, tag, wt, u, half = kinds(dtype)
    level = 1000.0 - np.arange(rows)[:, None] % 7 * 8.0  # steps of 0.5 (f16) and 4 (bf16) up to 1024
    v = np.repeat(level, n, axis=1)
    step = 0.5 if dtype == "f16" else 4.0
    v[np.arange(rows), np.arange(rows) % n] -= step
    x = laid(v, t)
    assert np.array_equal(wide64(x), v)
    y, mean, inv = forward(x, rows, n, tag, wt, 0.0)
    want, wm, wi = definition(v, 0.0)
    assert np.all(np.abs(inv - wi) <= 55 * u * wi)
    assert np.all(np.abs(mean - wm) <= 3 * u * np.abs(wm))
    assert np.all(np.abs(y - want) <= half * np.abs(want) + 110 * u * np.abs(want).max(axis=1, keepdims=True))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_constant_rows_have_no_deviation(gpu_lib, dtype):
    """epsilon alone decides: the mean of n equal numbers is off by at most 34 u of them, and what is left of
    the variance after its correction by 36 u of that square, far below epsilon = 1e-5 here."""
    t, tag, wt, u, half = kinds(dtype)
    levels = np.array([1000.0, -3.0, 60000.0, 0.0, -4096.0, 24.0, 0.5])
    rows, n = len(levels), 2000
    x = laid(np.repeat(levels[:, None], n, axis=1), t)
    y, mean, inv = forward(x, rows, n, tag, wt, 1e-5)
    level = wide64(x)[:, 0]
    left = 36 * u * (34 * u * np.abs(level)) ** 2
    assert np.all(left < 1e-7)
    wi = 1.0 / np.sqrt(1e-5)
    assert np.all(np.abs(inv - wi) <= (left / 1e-5 + 55 * u) * wi)
    assert np.all(np.abs(mean - level) <= 3 * u * np.abs(level))
    # a deviation is the difference of the first mean's error and its correction
    assert np.all(np.abs(y).max(axis=1) <= 36 * u * (34 * u * np.abs(level)) * wi * 2 + 1e-12)


@pytest.mark.parametrize("rows,n", [(2000, 4096), (100, 2001), (20, 20000)])
@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_means_near_zero(gpu_lib, dtype, rows, n):
    """Means of a fiftieth of the deviations.  The sum of the deviations reaches sqrt(n) and its last levels of
    additions leave about 2 * 2^-1 u sqrt(n) of it, sqrt(1 / n) u per entry or 50 / sqrt(n) u of the mean,
    whose own rounding is another half u: 1.6 u at n = 1000, in norm over the rows, and 4 u are allowed.
    Differences that share a rounding, half a step of u on average a quarter, would leave 12 u."""
    t, tag, wt, u, half = kinds(dtype)
    x = laid(inputs.normal(132, (rows, n)) + 0.02, t)
    y, mean, inv = forward(x, rows, n, tag, wt, 0.0)
    want, wm, wi = definition(wide64(x), 0.0)
    assert np.linalg.norm((mean - wm).astype(np.float64)) <= 4 * u * np.linalg.norm(wm.astype(np.float64))


@pytest.mark.parametrize("rows,n", [(40, 18000), (600, 16000), (100, 70000), (700, 6000)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_means_near_zero_of_16_bits(gpu_lib, dtype, rows, n):
    """Wide rows with means of a hundredth of the deviations.  Sums of 16-bit entries keep their 8 or 11 bits
    and the few of the count, so the first additions are exact and the last leave u sqrt(n) at most: with the
    mean's own rounding 100 / sqrt(n) + 1.5 u of the mean, 3 u in norm, and 4 u are allowed."""
    t, tag, wt, u, half = kinds(dtype)
    x = laid(2.0 * inputs.normal(133, (rows, n)) + 0.02, t)
    y, mean, inv = forward(x, rows, n, tag, wt, 0.0)
    want, wm, wi = definition(wide64(x), 0.0)
    assert np.linalg.norm((mean - wm).astype(np.float64)) <= 4 * u * np.linalg.norm(wm.astype(np.float64))
