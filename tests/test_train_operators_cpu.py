"""Argument checks of the training and serving operators, and their f64 definitions against finite
differences: everything that needs no GPU."""
import ctypes

import numpy as np
import pytest

import eshkol_b200 as eb
from eshkol_b200 import inputs
from oracle import operators_ref as ref


def test_the_calls_are_refused_without_a_device_and_compute_nothing():
    lib = eb.load_library()
    if lib.eshkol_gpu_init() == 1:
        pytest.skip("a GPU is present")
    a, out = np.ones((4, 4)), np.full((4, 4), 7.0)
    p, o = a.ctypes.data, out.ctypes.data
    assert lib.eshkol_b200_layernorm_forward_device(p, p, p, o, o, o, 4, 4, 0, 0, 1e-5, eb.DTYPE_F64) == -1
    assert lib.eshkol_b200_layernorm_gradients_device(p, p, p, p, p, o, o, o, 4, 4, 0, 0, 0, eb.DTYPE_F64) == -1
    assert lib.eshkol_b200_token_logprobs_device(p, None, None, o, o, None, None, 4, 4, 0, 0, eb.DTYPE_F64) == -1
    assert lib.eshkol_b200_token_logprobs_gradient_device(p, None, p, p, None, p, o, 4, 4, 0, 0, eb.DTYPE_F64) == -1
    assert (out == 7.0).all()
    with pytest.raises(RuntimeError):
        eb.layernorm_device(p, p, p, o, o, o, 4, 4, 1e-5, eb.DTYPE_F64)
    with pytest.raises(RuntimeError):
        eb.token_logprobs_device(p, 0, 0, o, o, 0, 0, 4, 4, 0, eb.DTYPE_F64)


def differences(f, x, step=1e-6):
    """gradient of the scalar f at x by central differences"""
    grad = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        keep = x[i]
        x[i] = keep + step
        up = f()
        x[i] = keep - step
        grad[i] = (up - f()) / (2 * step)
        x[i] = keep
    return grad


# central differences of step 1e-6 in f64: truncation below 1e-12 of third derivatives of order one,
# rounding 2^-53 * |f| / step, about 1e-9 for |f| of order ten
NEAR = 1e-7


def test_layernorm_gradients_against_differences():
    x, g = inputs.normal(41, (3, 5)), inputs.normal(42, (3, 5))
    gamma, beta = 1.0 + 0.2 * inputs.normal(43, (5,)), inputs.normal(44, (5,))

    def loss():
        return float((g * ref.layernorm_forward(x, gamma, beta, 1e-5)[0]).sum())

    _, mean, inv_std = ref.layernorm_forward(x, gamma, beta, 1e-5)
    gi, gg, gb = ref.layernorm_gradients(g, x, mean, inv_std, gamma)
    assert np.abs(gi - differences(loss, x)).max() < NEAR
    assert np.abs(gg - differences(loss, gamma)).max() < NEAR
    assert np.abs(gb - differences(loss, beta)).max() < NEAR


def test_token_logprob_gradient_against_differences():
    x = 2.0 * inputs.normal(45, (4, 7))
    x[1, 3] = -np.inf
    tokens = np.array([2, 0, -1, 6])
    g, h = inputs.normal(46, (4,)), inputs.normal(47, (4,))

    def loss():
        lp, ent = ref.token_logprobs(x, tokens, 0)[:2]
        return float((g * lp + h * ent).sum())

    _, ent, lse = ref.token_logprobs(x, tokens, 0)[:3]
    got = ref.token_logprobs_gradient(x, tokens, lse, ent, g, h)
    keep = x[1, 3]
    x[1, 3] = -1e3  # a difference needs a finite point; its probability is zero all the same
    want = differences(loss, x)
    x[1, 3] = keep
    assert np.abs(got - want).max() < NEAR


@pytest.mark.parametrize("act", [0, 1, 2])
def test_linear_gradients_against_differences(act):
    x, w, g = inputs.normal(81, (4, 6)), inputs.normal(82, (6, 5)), inputs.normal(83, (4, 5))
    bias = inputs.normal(84, (5,))

    def loss():
        return float((g * ref.linear_forward(x, w, bias, None, act)[0]).sum())

    pre = ref.linear_forward(x, w, bias, None, act)[1]
    assert np.abs(pre).min() > 1e-4  # no difference crosses ReLU's corner
    gx, gw, gb, _ = ref.linear_gradients(g, x, w, pre, act)
    assert np.abs(gx - differences(loss, x)).max() < 10 * NEAR
    assert np.abs(gw - differences(loss, w)).max() < 10 * NEAR
    assert np.abs(gb - differences(loss, bias)).max() < 10 * NEAR


def test_linear_calls_are_refused_without_a_device():
    lib = eb.load_library()
    if lib.eshkol_gpu_init() == 1:
        pytest.skip("a GPU is present")
    a, out = np.ones((4, 4), dtype=np.float32), np.full((4, 4), 7.0, dtype=np.float32)
    p, o = a.ctypes.data, out.ctypes.data
    opts = eb.make_linear_opts(eb.DTYPE_F32)
    assert ctypes.sizeof(opts) == 80
    assert lib.eshkol_b200_linear_forward_device(p, p, o, 4, 4, 4, ctypes.byref(opts)) == -1
    assert lib.eshkol_b200_linear_gradients_device(p, p, p, o, o, o, 4, 4, 4, ctypes.byref(opts)) == -1
    assert (out == 7.0).all()
    with pytest.raises(RuntimeError):
        eb.linear_device(p, p, o, 4, 4, 4, opts)
