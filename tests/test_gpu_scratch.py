"""Scratch of the training and serving operators: calls of several host threads, and calls that need none."""
import threading

import numpy as np
import pytest

import eshkol_b200 as eb
from eshkol_b200 import inputs
from test_gpu_norm_logprobs import done, kinds, laid, room, vector, wide64

pytestmark = pytest.mark.gpu


def linear_case(seed, dtype, rows, k, n):
    """all gradients of a layer whose operands and dz are packed or split into scratch"""
    t, tag, wt, u, half = kinds(dtype)
    x, w = laid(inputs.normal(seed, (rows, k)), t, 3, 1), laid(inputs.normal(seed + 1, (k, n)) / np.sqrt(k), t, 3, 1)
    g, z = laid(inputs.normal(seed + 2, (rows, n)), t, 3, 1), laid(inputs.normal(seed + 3, (rows, n)), t, 3, 1)
    outs = [room((rows, k), t, 3, 1), room((k, n), t, 3, 1), room((n,), wt)]
    opts = eb.make_linear_opts(tag, activation=2, pre=z.data_ptr(), ldx=x.stride(0), ldw=w.stride(0), ldy=g.stride(0), ld_pre=z.stride(0))
    keep = (x, w, g, z, opts)
    return lambda: eb.linear_gradients_device(keep[2].data_ptr(), keep[0].data_ptr(), keep[1].data_ptr(), *(o.data_ptr() for o in outs),
                                              rows, k, n, opts), outs


def norm_case(seed, dtype, rows, n):
    """gradients of a norm whose weight gradients are joined from scratch"""
    t, tag, wt, u, half = kinds(dtype)
    x, g = laid(inputs.normal(seed, (rows, n)), t), laid(inputs.normal(seed + 1, (rows, n)), t)
    mean, inv = vector(np.zeros(rows), wt), vector(np.ones(rows), wt)
    outs = [room((rows, n), t), room((n,), wt), room((n,), wt)]
    keep = (x, g, mean, inv)
    return lambda: eb.layernorm_gradients_device(keep[1].data_ptr(), keep[0].data_ptr(), keep[2].data_ptr(), keep[3].data_ptr(), 0,
                                                 *(o.data_ptr() for o in outs), rows, n, tag), outs


def test_two_host_threads(gpu_lib):
    """Two threads make calls of different and growing sizes, each into its own results: the bits are those
    of the same calls made one after the other."""
    import torch
    mine = [linear_case(151, "f32", 70, 130, 90), norm_case(155, "f32", 300, 600), linear_case(157, "f16", 333, 401, 599),
            linear_case(161, "f32", 900, 700, 1100)]
    others = [norm_case(165, "f64", 200, 333), linear_case(167, "bf16", 257, 301, 203), linear_case(171, "f32", 520, 333, 777),
              linear_case(175, "f16", 1500, 1001, 1203)]
    want = []
    for call, outs in mine + others:
        call()
        done()
        want.append([wide64(o) for o in outs])
    for turn in range(3):
        for _, outs in mine + others:
            for o in outs:
                o.fill_(float("nan"))
        torch.cuda.synchronize()
        start, errors = threading.Barrier(2), []

        def work(cases):
            try:
                start.wait(timeout=30)
                for _ in range(20):
                    for call, _ in cases:
                        call()
            except Exception as e:  # reported by the test's own thread
                errors.append(e)

        threads = [threading.Thread(target=work, args=(c,)) for c in (mine, others)]
        for th in threads:
            th.start()
        for th in threads:
            th.join(timeout=60)
        assert not errors and not any(th.is_alive() for th in threads)
        done()
        for (_, outs), w in zip(mine + others, want):
            assert all(np.array_equal(wide64(o), v) for o, v in zip(outs, w))
