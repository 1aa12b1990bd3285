"""The linear layer and its gradients on the GPU against their f64 definitions on the stored inputs.

Tolerances: products of 16-bit numbers are exact in f32; the tensor core adds 16 of them and the running
sum per step with f32 truncation, so a sum over K is off by at most (K / 16 + 32) 2^-23 of the sum of the
terms' magnitudes S (f32 operands: six products of parts, 6 K / 16 steps).  The activations pass an error
on with a slope of at most 1.13 and add 2^-18 of their own; a result is rounded to its type once (half)."""
import ctypes

import numpy as np
import pytest

import eshkol_b200 as eb
from eshkol_b200 import api, inputs
from oracle import operators_ref as ref
from test_gpu_norm_logprobs import done, kinds, laid, room, untouched, vector, wide64

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1, 0, 0), (3, 5, 7, 0, 0), (1, 64, 64, 0, 0), (1, 4096, 304, 0, 0), (17, 1001, 999, 0, 0),
          (128, 256, 512, 0, 0), (130, 300, 520, 8, 8), (257, 1000, 136, 5, 3), (300, 2048, 2048, 0, 0),
          (64, 8192, 192, 0, 0), (700, 96, 40, 16, 8), (1000, 72, 1100, 1, 1), (2, 640, 384, 0, 0), (4, 1000, 520, 0, 0),
          (8, 1030, 514, 1, 1), (12, 600, 250, 0, 0), (40, 90, 254, 2, 2), (520, 520, 1040, 0, 0)]


def steps(k, dtype):
    return ((6 if dtype == "f32" else 1) * k / 16 + 32) * 2.0 ** -23


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k,n,pad,offset", SHAPES)
@pytest.mark.parametrize("act,trans_w", [(0, False), (1, True), (2, False), (2, True)])
def test_linear(gpu_lib, dtype, rows, k, n, pad, offset, act, trans_w):
    t, tag, wt, u, half = kinds(dtype)
    x = laid(inputs.normal(91, (rows, k)), t, pad, offset)
    w_np = inputs.normal(92, (k, n)) / np.sqrt(k)
    w = laid(w_np.T if trans_w else w_np, t, pad, offset)
    bias, res = vector(0.3 * inputs.normal(93, (n,)), t), laid(inputs.normal(94, (rows, n)), t, pad, offset)
    y, pre = room((rows, n), t, pad, offset), room((rows, n), t, pad, offset)

    def call(out, b, r, z):
        opts = eb.make_linear_opts(tag, activation=act, trans_w=trans_w, bias=b.data_ptr() if b is not None else 0,
                                   residual=r.data_ptr() if r is not None else 0, pre=z.data_ptr() if z is not None else 0,
                                   ldx=x.stride(0), ldw=w.stride(0), ldy=out.stride(0), ld_residual=r.stride(0) if r is not None else 0,
                                   ld_pre=z.stride(0) if z is not None else 0)
        eb.linear_device(x.data_ptr(), w.data_ptr(), out.data_ptr(), rows, k, n, opts)
        done()

    call(y, bias, res, pre)
    xs, ws, bs, rs = wide64(x), wide64(w), wide64(bias), wide64(res)
    ws = ws.T if trans_w else ws
    want, wz = ref.linear_forward(xs, ws, bs, rs, act)
    err = steps(k, dtype) * (np.abs(xs) @ np.abs(ws) + np.abs(bs))
    # f16: below its normal numbers the step is fixed
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0
    assert np.all(np.abs(wide64(pre) - wz) <= half * np.abs(wz) + (1 + half) * err + tiny)
    own = 2.0 ** -18 * np.abs(wz) if act == 2 else 0.0
    assert np.all(np.abs(wide64(y) - want) <= half * np.abs(want) + (1 + half) * (1.13 * err + own + 2 * u * np.abs(want)) + tiny)
    assert untouched(y, offset) and untouched(pre, offset)
    # bare, and with the residual in place of the result
    bare = room((rows, n), t, pad, offset)
    call(bare, None, None, None)
    want0, wz0 = ref.linear_forward(xs, ws, None, None, act)
    own0 = 2.0 ** -18 * np.abs(wz0) if act == 2 else 0.0
    assert np.all(np.abs(wide64(bare) - want0) <= half * np.abs(want0) + (1 + half) * (1.13 * err + own0) + tiny)
    call(res, bias, res, None)
    assert np.array_equal(wide64(res), wide64(y))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k,n,pad,offset", SHAPES)
@pytest.mark.parametrize("act,trans_w", [(0, True), (1, False), (2, True)])
def test_linear_gradients(gpu_lib, dtype, rows, k, n, pad, offset, act, trans_w):
    t, tag, wt, u, half = kinds(dtype)
    x = laid(inputs.normal(95, (rows, k)), t, pad, offset)
    w_np = inputs.normal(96, (k, n)) / np.sqrt(k)
    w = laid(w_np.T if trans_w else w_np, t, pad, offset)
    g, z = laid(inputs.normal(97, (rows, n)), t, pad, offset), laid(2.0 * inputs.normal(98, (rows, n)), t, pad, offset)
    gx, gw, gb = room((rows, k), t, pad, offset), room(tuple(w.shape), t, pad, offset), room((n,), wt)
    opts = eb.make_linear_opts(tag, activation=act, trans_w=trans_w, pre=z.data_ptr() if act else 0, ldx=x.stride(0),
                               ldw=w.stride(0), ldy=g.stride(0), ld_pre=z.stride(0))

    def call(a, b, c):
        eb.linear_gradients_device(g.data_ptr(), x.data_ptr() if b is not None else 0, w.data_ptr() if a is not None else 0,
                                   a.data_ptr() if a is not None else 0, b.data_ptr() if b is not None else 0,
                                   c.data_ptr() if c is not None else 0, rows, k, n, opts)
        done()

    call(gx, gw, gb)
    xs, ws, gs, zs = wide64(x), wide64(w), wide64(g), wide64(z)
    ws = ws.T if trans_w else ws
    wx, ww, wb, dz = ref.linear_gradients(gs, xs, ws, zs, act)
    got_w = wide64(gw).T if trans_w else wide64(gw)
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0
    # dz is rounded to the storage type for the products (f32: not at all) where there is an activation
    rounded = (half if act and dtype != "f32" else 0.0) + (2.0 ** -17 if act == 2 else 0.0)
    off = rounded * np.abs(gs) + tiny
    tol_x = half * np.abs(wx) + (1 + half) * (off @ np.abs(ws).T + steps(n, dtype) * (np.abs(dz) + off) @ np.abs(ws).T) + tiny
    tol_w = half * np.abs(ww) + (1 + half) * (np.abs(xs).T @ off + steps(rows, dtype) * np.abs(xs).T @ (np.abs(dz) + off)) + tiny
    assert np.all(np.abs(wide64(gx) - wx) <= 1.13 * tol_x)
    assert np.all(np.abs(got_w - ww) <= 1.13 * tol_w)
    # column sums: at most rows / 8 additions by a warp, eight warps, a few hundred blocks
    assert np.all(np.abs(wide64(gb) - wb) <= ((rows / 8 + 300) * u + (2.0 ** -17 if act == 2 else 0.0)) * np.abs(gs).sum(axis=0))
    assert untouched(gx, offset) and untouched(gw, offset)
    first = [wide64(v) for v in (gx, gw, gb)]
    for v in (gx, gw, gb):
        v.fill_(float("nan"))
    import torch
    torch.cuda.synchronize()
    call(gx, gw, gb)
    assert all(np.array_equal(a, wide64(b)) for a, b in zip(first, (gx, gw, gb)))  # the same bits again
    # one at a time: the sums may be cut differently, the results stay within their tolerances
    for v in (gx, gw, gb):
        v.fill_(float("nan"))
    torch.cuda.synchronize()
    call(gx, None, None)
    assert np.all(np.abs(wide64(gx) - wx) <= 1.13 * tol_x)
    call(None, gw, None)
    assert np.all(np.abs((wide64(gw).T if trans_w else wide64(gw)) - ww) <= 1.13 * tol_w)
    call(None, None, gb)
    assert np.array_equal(wide64(gb), first[2])


def test_small_integers_are_exact(gpu_lib):
    """Sums of integers that f32 and the storage types hold have no rounding at all, whatever the tiling."""
    for dtype in ("f32", "f16", "bf16"):
        t, tag, wt, u, half = kinds(dtype)
        for rows, k, n in ((1, 7, 9), (200, 320, 640), (129, 130, 700), (5, 3000, 65)):
            a = np.rint(inputs.uniform(99, (rows, k)) * 1.49)
            b = np.rint(inputs.uniform(100, (k, n)) * 1.49)
            if dtype != "f32":
                a[:, 100:] = 0.0  # keeps the sums within the integers of bf16
            x, w, y = laid(a, t), laid(b, t), room((rows, n), t)
            eb.linear_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), rows, k, n, eb.make_linear_opts(tag))
            done()
            assert np.array_equal(wide64(y), a @ b)


def test_special_values_stay_in_their_rows(gpu_lib):
    """NaN or infinity in a row of x reaches that row of y and no other, and a padded batch's rows behind
    the last one are left alone."""
    t, tag, wt, u, half = kinds("bf16")
    xv = inputs.normal(101, (50, 200))
    xv[7, 3], xv[9, 5] = np.nan, np.inf
    x, w = laid(xv, t), laid(inputs.normal(102, (200, 130)), t)
    y = room((64, 130), t, fill=5.0)
    eb.linear_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), 50, 200, 130, eb.make_linear_opts(tag))
    done()
    got = wide64(y)
    assert np.isnan(got[7]).all() and not np.isfinite(got[9]).any()
    keep = [r for r in range(50) if r not in (7, 9)]
    assert np.isfinite(got[keep]).all() and (got[50:] == 5.0).all()


def test_products_of_two_rounds_and_more(gpu_lib):
    """More tiles than SMs in both products of the gradients, unevenly: every tile is written once."""
    import torch
    t, tag, wt, u, half = kinds("bf16")
    rows, k, n = 2100, 2300, 4200
    x, w, g = (torch.randint(-1, 2, s, device="cuda").to(t) for s in ((rows, k), (k, n), (rows, n)))
    x[:, 60:] = 0  # keeps the sums within the integers of bf16
    g[:, 60:] = 0
    g[60:] = 0
    gx, gw, y = room((rows, k), t), room((k, n), t), room((rows, n), t)
    eb.linear_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), rows, k, n, eb.make_linear_opts(tag))
    eb.linear_gradients_device(g.data_ptr(), x.data_ptr(), w.data_ptr(), gx.data_ptr(), gw.data_ptr(), 0, rows, k, n, eb.make_linear_opts(tag))
    done()
    f = [v.to(torch.float64) for v in (x, w, g)]
    assert torch.equal(y.to(torch.float64), f[0] @ f[1])
    assert torch.equal(gx.to(torch.float64), f[2] @ f[1].T)
    assert torch.equal(gw.to(torch.float64), f[0].T @ f[2])


def test_gelu_far_out(gpu_lib):
    """Far from zero the activation is the identity or zero and its slope one or zero: no overflow on the way."""
    for dtype in ("f32", "bf16"):
        t, tag, wt, u, half = kinds(dtype)
        z = np.array([[-1e30, -3e4, -30.0, -0.0, 0.0, 30.0, 3e4, 1e30]])
        x, w = laid(np.ones((1, 1)), t), laid(z, t)
        y = room((1, 8), t)
        eb.linear_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), 1, 1, 8, eb.make_linear_opts(tag, activation=2))
        done()
        assert np.array_equal(wide64(y), np.where(wide64(w) > 0, wide64(w), 0.0))
        g, pre, gb = laid(np.ones((1, 8)), t), laid(z, t), room((8,), wt)
        eb.linear_gradients_device(g.data_ptr(), 0, 0, 0, 0, gb.data_ptr(), 1, 1, 8,
                                   eb.make_linear_opts(tag, activation=2, pre=pre.data_ptr()))
        done()
        assert np.array_equal(wide64(gb), [0, 0, 0, 0.5, 0.5, 1, 1, 1])


def test_refusals_and_empty_calls(gpu_lib):
    import torch
    lib = gpu_lib
    t = torch.float32
    x, w, y = room((4, 8), t, fill=1.0), room((8, 6), t, fill=1.0), room((4, 6), t, fill=7.0)
    p, q, o = x.data_ptr(), w.data_ptr(), y.data_ptr()
    fwd, bwd = lib.eshkol_b200_linear_forward_device, lib.eshkol_b200_linear_gradients_device

    def opts(**kw):
        return ctypes.byref(eb.make_linear_opts(kw.pop("dtype", eb.DTYPE_F32), **kw))

    assert fwd(p, q, o, 4, 8, 6, None) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(dtype=eb.DTYPE_F64)) == -1          # the f64 products serve that
    assert fwd(p, q, o, 4, 8, 6, opts(dtype=4)) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(activation=3)) == -1
    assert fwd(p, q, o, 4, 0, 6, opts()) == -1
    assert fwd(p, q, o, 4, 8, 0, opts()) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(ldx=7)) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(ldw=5)) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(ldw=6, trans_w=True)) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(ldy=-1)) == -1
    assert fwd(None, q, o, 4, 8, 6, opts()) == -1
    assert fwd(p, q, p, 4, 8, 6, opts()) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(pre=o)) == -1
    assert fwd(p, q, o, 4, 8, 6, opts(residual=o, ld_residual=7)) == -1
    assert fwd(p, q, o, 1 << 31, 8, 6, opts()) == -1
    assert bwd(o, p, q, None, None, None, 4, 8, 6, opts()) == -1          # nothing asked for
    assert bwd(o, p, None, p + 4096, None, None, 4, 8, 6, opts()) == -1   # w missing
    assert bwd(o, None, q, None, q + 4096, None, 4, 8, 6, opts()) == -1   # x missing
    assert bwd(o, p, q, p, None, None, 4, 8, 6, opts()) == -1             # over an input
    assert bwd(o, p, q, None, q, None, 4, 8, 6, opts()) == -1
    assert bwd(o, p, q, None, None, q, 4, 8, 6, opts(activation=2)) == -1  # pre missing
    done()
    assert bool((y == 7.0).all())
    # no rows: y is empty, the sums are zero and the pitch's gap is left alone
    assert fwd(None, q, None, 0, 8, 6, opts()) == 0
    gw, gb = room((8, 6), t, 2, 1), room((6,), t)
    assert bwd(None, None, None, None, gw.data_ptr(), gb.data_ptr(), 0, 8, 6, opts(ldw=8)) == 0
    done()
    assert bool((gw == 0).all()) and bool((gb == 0).all()) and untouched(gw, 1)


def test_a_wait_that_runs_out_is_reported_once(gpu_lib):
    """The producer withholds one stage (a host-side switch): the bounded waits end the kernel, the status
    is reported, and the next call is right."""
    t, tag, wt, u, half = kinds("bf16")
    x, w, y = laid(np.ones((128, 256)), t), laid(np.ones((256, 64)), t), room((128, 64), t)
    lib = gpu_lib
    lib.eshkol_b200_debug_set_wait_limit_ns(1_000_000)
    lib.eshkol_b200_debug_withhold_arrival(1)
    try:
        assert lib.eshkol_b200_linear_forward_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), 128, 256, 64,
                                                     ctypes.byref(eb.make_linear_opts(tag))) == 0
        assert api.sync_status() > 0
    finally:
        lib.eshkol_b200_debug_set_wait_limit_ns(0)
        lib.eshkol_b200_debug_withhold_arrival(0)
    eb.linear_device(x.data_ptr(), w.data_ptr(), y.data_ptr(), 128, 256, 64, eb.make_linear_opts(tag))
    done()
    assert bool((y == 256.0).all())


def test_a_training_step_of_a_block(gpu_lib):
    """norm -> up (GELU) -> down (+ residual) -> norm -> logits -> log probabilities, and all gradients back,
    eager and as a captured graph, against the same chain in f64 on the stored tensors of each step."""
    import torch
    t, tag, wt, u, half = kinds("f32")
    rows, d, ff, v = 96, 136, 520, 1003
    stream = torch.cuda.ExternalStream(api.stream_handle())

    def P(x):
        return x.data_ptr()

    x0 = laid(inputs.normal(111, (rows, d)), t)
    g1, b1, g2, b2 = (vector(s + 0.1 * inputs.normal(112 + i, (d,)), t) for i, s in enumerate((1.0, 0.0, 1.0, 0.0)))
    w1, w2, we = (laid(inputs.normal(116 + i, s) / np.sqrt(s[j]), t) for i, (s, j) in
                  enumerate((((d, ff), 0), ((ff, d), 0), ((v, d), 1))))
    c1, c2 = vector(0.1 * inputs.normal(119, (ff,)), t), vector(0.1 * inputs.normal(120, (d,)), t)
    tokens_np = (np.arange(rows) * 17) % v
    tokens_np[::7] = -1
    tokens = torch.from_numpy(tokens_np).cuda()
    glp, gent = vector(-np.ones(rows) / rows, wt), vector(-0.01 * np.ones(rows), wt)
    R = lambda *s: room(s, t)  # noqa: E731
    h, m1, i1, a, z, y, h2, m2, i2, logit = (R(rows, d), R(rows), R(rows), R(rows, ff), R(rows, ff), R(rows, d), R(rows, d),
                                             R(rows), R(rows), R(rows, v))
    lp, ent, lse = R(rows), R(rows), R(rows)
    glogit, gh2, gwe, gy, gg2, gb2, ga, gw2, gc2, gh, gw1, gc1, gx, gg1, gb1 = (
        R(rows, v), R(rows, d), R(v, d), R(rows, d), R(d), R(d), R(rows, ff), R(ff, d), R(d), R(rows, d), R(d, ff), R(ff),
        R(rows, d), R(d), R(d))

    def step():
        eb.layernorm_device(P(x0), P(g1), P(b1), P(h), P(m1), P(i1), rows, d, 1e-5, tag)
        eb.linear_device(P(h), P(w1), P(a), rows, d, ff, eb.make_linear_opts(tag, activation=2, bias=P(c1), pre=P(z)))
        eb.linear_device(P(a), P(w2), P(y), rows, ff, d, eb.make_linear_opts(tag, bias=P(c2), residual=P(x0)))
        eb.layernorm_device(P(y), P(g2), P(b2), P(h2), P(m2), P(i2), rows, d, 1e-5, tag)
        eb.linear_device(P(h2), P(we), P(logit), rows, d, v, eb.make_linear_opts(tag, trans_w=True))
        eb.token_logprobs_device(P(logit), P(tokens), P(lp), P(ent), P(lse), 0, 0, rows, v, 0, tag)
        eb.token_logprobs_gradient_device(P(logit), P(tokens), P(lse), P(ent), P(glp), P(gent), P(glogit), rows, v, tag)
        eb.linear_gradients_device(P(glogit), P(h2), P(we), P(gh2), P(gwe), 0, rows, d, v, eb.make_linear_opts(tag, trans_w=True))
        eb.layernorm_gradients_device(P(gh2), P(y), P(m2), P(i2), P(g2), P(gy), P(gg2), P(gb2), rows, d, tag)
        eb.linear_gradients_device(P(gy), P(a), P(w2), P(ga), P(gw2), P(gc2), rows, ff, d, eb.make_linear_opts(tag))
        eb.linear_gradients_device(P(ga), P(h), P(w1), P(gh), P(gw1), P(gc1), rows, d, ff,
                                   eb.make_linear_opts(tag, activation=2, pre=P(z)))
        eb.layernorm_gradients_device(P(gh), P(x0), P(m1), P(i1), P(g1), P(gx), P(gg1), P(gb1), rows, d, tag)

    outs = [lp, ent, glogit, gwe, gg2, gb2, gw2, gc2, gw1, gc1, gx, gg1, gb1]
    step()
    done()
    eager = [wide64(o) for o in outs]
    # the chain in f64
    X, W1, W2, WE = wide64(x0), wide64(w1), wide64(w2), wide64(we).T
    H, M1, I1 = ref.layernorm_forward(X, wide64(g1), wide64(b1), 1e-5)
    A, Z = ref.linear_forward(H, W1, wide64(c1), None, 2)
    Y, _ = ref.linear_forward(A, W2, wide64(c2), X, 0)
    H2, M2, I2 = ref.layernorm_forward(Y, wide64(g2), wide64(b2), 1e-5)
    L = H2 @ WE
    LP, ENT, LSE = ref.token_logprobs(L, tokens_np, 0)[:3]
    GL = ref.token_logprobs_gradient(L, tokens_np, LSE, ENT, wide64(glp), wide64(gent))
    GH2, GWE, _, _ = ref.linear_gradients(GL, H2, WE, None, 0)
    GY, GG2, GB2 = ref.layernorm_gradients(GH2, Y, M2, I2, wide64(g2))
    GA, GW2, GC2, _ = ref.linear_gradients(GY, A, W2, None, 0)
    GH, GW1, GC1, _ = ref.linear_gradients(GA, H, W1, Z, 2)
    GX, GG1, GB1 = ref.layernorm_gradients(GH, X, M1, I1, wide64(g1))
    want = [LP, ENT, GL, GWE.T, GG2, GB2, GW2, GC2, GW1, GC1, GX, GG1, GB1]
    # twelve steps of f32, each off by at most a few hundred u of its terms' magnitudes and none of them
    # badly conditioned here: 1e-4 of the result's norm
    for got, w in zip(eager, want):
        assert np.linalg.norm(got - w) <= 1e-4 * np.linalg.norm(w)
    for o in outs:
        o.fill_(float("nan"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    done()
    assert all(np.array_equal(a, wide64(b)) for a, b in zip(eager, outs))
