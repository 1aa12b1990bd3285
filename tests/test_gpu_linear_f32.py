"""The accuracy of the linear layer's f32 products beyond a few rows, where they are made of bf16 parts.

Norm: within a hand-over the running sum of 256 terms goes through 16 truncated additions.  With terms of
size s the sum after j of them is about 0.8 * 4 sqrt(j) s, and truncation takes 0.75 * 2^-24 of it on average
(half a step, steps between 2^-24 and 2^-23): 0.75 * 137 * 2^-24 s per hand-over whose sum is 16 s, which is
3.8e-7 of the norm.  Products left out (2^-24 of a term at worst) and the roundings of the hand-overs' sums
stay below a tenth of that.  A bound of 6e-7; a missing part costs 3.5e-6 (tests/test_f32_parts_cpu.py),
hand-overs eight times as long 2e-6."""
import numpy as np
import pytest

import eshkol_b200 as eb
from eshkol_b200 import inputs
from test_gpu_norm_logprobs import done, kinds, laid, room, wide64

pytestmark = pytest.mark.gpu
NORM = 6e-7


def forward(x, w, rows, k, n, trans_w):
    t, tag, wt, u, half = kinds("f32")
    y = room((rows, n), t)
    eb.linear_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), rows, k, n,
                     eb.make_linear_opts(tag, trans_w=trans_w, ldx=x.stride(0), ldw=w.stride(0)))
    done()
    return wide64(y)


def gradients(g, x, w, rows, k, n, trans_w):
    t, tag, wt, u, half = kinds("f32")
    gx, gw = room((rows, k), t), room((n, k) if trans_w else (k, n), t)
    eb.linear_gradients_device(g.data_ptr(), x.data_ptr(), w.data_ptr(), gx.data_ptr(), gw.data_ptr(), 0, rows, k, n,
                               eb.make_linear_opts(tag, trans_w=trans_w))
    done()
    return wide64(gx), wide64(gw).T if trans_w else wide64(gw)


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("rows,k,n", [(64, 8192, 192), (300, 2048, 2048), (777, 2001, 1603), (2500, 1030, 2100), (17, 5000, 4000)])
@pytest.mark.parametrize("trans_w", [False, True])
def test_the_error_in_norm(gpu_lib, rows, k, n, trans_w):
    t = kinds("f32")[0]
    x, wv, g = (inputs.normal(191 + i, s) for i, s in enumerate(((rows, k), (k, n), (rows, n))))
    x, w, g = laid(x, t), laid(wv.T if trans_w else wv, t), laid(g, t)
    xs, gs, ws = wide64(x), wide64(g), wide64(w).T if trans_w else wide64(w)
    assert off(forward(x, w, rows, k, n, trans_w), xs @ ws) <= NORM
    gx, gw = gradients(g, x, w, rows, k, n, trans_w)
    assert off(gx, gs @ ws.T) <= NORM
    if rows > 17:
        assert off(gw, xs.T @ gs) <= NORM


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("exponent", [-103, -20, 0, 90])
def test_all_24_bits_of_both_operands_arrive(gpu_lib, exponent, trans_w):
    """One operand of full significands, the other with a single power of two to every result: each result
    is one operand's value, scaled, and needs all its parts."""
    t = kinds("f32")[0]
    rows, k, n = 150, 700, 330
    full = lambda seed, s: ((1.0 + np.abs(inputs.uniform(seed, s))).clip(1.0, 1.9999) * 2.0 ** exponent).astype(np.float32).astype(np.float64)  # noqa: E731

    def single(outer, inner):  # one entry in every column
        m = np.zeros((outer, inner))
        m[(np.arange(inner) * 37) % outer, np.arange(inner)] = 2.0 ** (np.arange(inner) % 9)
        return m

    lay = lambda m: laid(m.T if trans_w else m, t)  # noqa: E731
    x, w = full(194, (rows, k)), single(k, n)
    assert np.array_equal(forward(laid(x, t), lay(w), rows, k, n, trans_w), x @ w)
    x, w = single(k, rows).T.copy(), full(195, (k, n))
    assert np.array_equal(forward(laid(x, t), lay(w), rows, k, n, trans_w), x @ w)
    # gradients: grad_x = g w^T, grad_w = x^T g
    x, w, g = single(rows, k), single(n, k).T.copy(), full(196, (rows, n))
    gx, gw = gradients(laid(g, t), laid(x, t), lay(w), rows, k, n, trans_w)
    assert np.array_equal(gx, g @ w.T) and np.array_equal(gw, x.T @ g)


@pytest.mark.parametrize("rows", [1, 12, 16, 17, 200])
@pytest.mark.parametrize("trans_w", [False, True])
def test_infinities_and_the_largest_numbers_stay_in_their_rows(gpu_lib, rows, trans_w):
    """Infinity: no finite result in its row (few rows: infinity, else NaN) and no trace in another.  Up to
    3.38e38 numbers are multiplied like any others."""
    t, tag, wt, u, half = kinds("f32")
    k, n = 300, 130
    x, wv = inputs.normal(197, (rows, k)), np.abs(inputs.normal(198, (k, n))) + 0.5
    clean = laid(x, t)
    w = laid(wv.T if trans_w else wv, t)
    at = rows // 2
    x[at, 7] = np.inf
    got, ref = forward(laid(x, t), w, rows, k, n, trans_w), forward(clean, w, rows, k, n, trans_w)
    assert not np.isfinite(got[at]).any()
    keep = np.arange(rows) != at
    assert np.array_equal(got[keep], ref[keep])
    x[:] = 0.0
    x[at, 7] = 3.38e38
    wv[:] = 2.0 ** -3
    got = forward(laid(x, t), laid(wv.T if trans_w else wv, t), rows, k, n, trans_w)
    assert np.array_equal(got[at], np.full(n, np.float64(np.float32(3.38e38)) / 8)) and (got[keep] == 0).all()
