"""Layer norm and token log probabilities on the GPU against their f64 definitions
(oracle/operators_ref.py) on the stored inputs.

Tolerances: u is the rounding of the stat type (2^-24, or 2^-53 for f64 tensors), a result is rounded to
its storage type once (half a step: eps / 2).  A thread adds at most 64 values before the shuffles, so a
sum of n terms is off by at most 80 u times the sum of their magnitudes; an inverse deviation takes that
once more, and the products a few u: 200 u of the magnitudes involved covers a whole expression."""
import numpy as np
import pytest

import eshkol_b200 as eb
from eshkol_b200 import api, inputs
from oracle import operators_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = ["f64", "f32", "f16", "bf16"]


def kinds(name):
    import torch
    t = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]
    tag = {"f64": eb.DTYPE_F64, "f32": eb.DTYPE_F32, "f16": eb.DTYPE_F16, "bf16": eb.DTYPE_BF16}[name]
    wide = torch.float64 if name == "f64" else torch.float32
    u = 2.0 ** -53 if name == "f64" else 2.0 ** -24
    return t, tag, wide, u, torch.finfo(t).eps / 2


def laid(values, t, pad=0, offset=0):
    """values in rows of a wider buffer of NaN, `offset` elements in; complete before the library reads it"""
    import torch
    v = torch.from_numpy(np.ascontiguousarray(values)).cuda().to(t)
    buf = torch.full((v.shape[0], v.shape[1] + pad), float("nan"), dtype=t, device="cuda")
    view = buf[:, offset:offset + v.shape[1]]
    view.copy_(v)
    torch.cuda.synchronize()
    return view


def vector(values, t):
    import torch
    v = torch.from_numpy(np.ascontiguousarray(values)).cuda().to(t)
    torch.cuda.synchronize()
    return v


def room(shape, t, pad=0, offset=0, fill=None):
    import torch
    fill = float("nan") if fill is None else fill
    if len(shape) == 1:
        b = torch.full(shape, fill, dtype=t, device="cuda")
    else:
        b = torch.full((shape[0], shape[1] + pad), fill, dtype=t, device="cuda")[:, offset:offset + shape[1]]
    torch.cuda.synchronize()
    return b


def wide64(t):
    import torch
    return t.to(torch.float64).cpu().numpy()


def done():
    assert api.sync_status() == 0


def untouched(view, offset):
    """the elements around the rows of a result of room(..., pad) are still NaN"""
    import torch
    base = view._base if view._base is not None else view
    keep = torch.ones(base.shape[1], dtype=torch.bool, device=base.device)
    keep[offset:offset + view.shape[1]] = False
    return bool(torch.isnan(base[:, keep]).all())


SHAPES = [(1, 1, 0, 0), (1, 4096, 0, 0), (3, 7, 0, 0), (1000, 40, 8, 8), (37, 1000, 0, 0), (130, 1001, 6, 1),
          (2000, 256, 0, 0), (5, 5000, 3, 2), (700, 2048, 0, 0), (3, 20000, 0, 0), (150, 9001, 0, 0), (2, 70000, 1, 1),
          (900, 810, 0, 0), (70, 5678, 2, 2), (640, 16390, 0, 0), (1300, 130, 1, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,pad,offset", SHAPES)
def test_layernorm(gpu_lib, dtype, rows, n, pad, offset):
    t, tag, wt, u, half = kinds(dtype)
    x = laid(inputs.normal(51, (rows, n)) * 3.0 + 1.5, t, pad, offset)
    gamma, beta = vector(1.0 + 0.3 * inputs.normal(52, (n,)), t), vector(inputs.normal(53, (n,)), t)
    y, mean, inv = room((rows, n), t, pad, offset), room((rows,), wt), room((rows,), wt)
    eb.layernorm_device(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), mean.data_ptr(), inv.data_ptr(),
                        rows, n, 1e-5, tag, ldx=x.stride(0), ldy=y.stride(0))
    done()
    xs, gs, bs = wide64(x), wide64(gamma), wide64(beta)
    want, wm, wi = ref.layernorm_forward(xs, gs, bs, 1e-5)
    xhat = np.abs((xs - wm[:, None]) * wi[:, None])
    tol = half * np.abs(want) + 200 * u * (xhat.max(axis=1, keepdims=True) * np.abs(gs) + np.abs(bs))
    assert np.all(np.abs(wide64(y) - want) <= tol)
    assert np.all(np.abs(wide64(mean) - wm) <= 200 * u * np.abs(xs).max(axis=1))
    assert np.all(np.abs(wide64(inv) - wi) <= 200 * u * wi)
    assert untouched(y, offset)
    # without weights and statistics, in place
    again = laid(wide64(x), t, pad, offset)
    eb.layernorm_device(again.data_ptr(), 0, 0, again.data_ptr(), 0, 0, rows, n, 1e-5, tag, ldx=again.stride(0),
                        ldy=again.stride(0))
    done()
    want = ref.layernorm_forward(xs, None, None, 1e-5)[0]
    assert np.all(np.abs(wide64(again) - want) <= half * np.abs(want) + 200 * u * xhat.max(axis=1, keepdims=True))


def test_layernorm_of_rows_far_from_zero(gpu_lib):
    """mean 1000 times the deviation: the deviations' own sum takes the rounding of the mean out."""
    t, tag, wt, u, half = kinds("f32")
    x = laid(inputs.normal(54, (60, 4099)) + 1000.0, t)
    y = room(x.shape, t)
    eb.layernorm_device(x.data_ptr(), 0, 0, y.data_ptr(), 0, 0, 60, 4099, 0.0, tag)
    done()
    want = ref.layernorm_forward(wide64(x), None, None, 0.0)[0]
    assert np.all(np.abs(wide64(y) - want) <= 200 * u * np.abs(want).max(axis=1, keepdims=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,pad,offset", SHAPES + [(5000, 33, 0, 0), (20000, 16, 0, 0), (600, 8192, 0, 0)])
def test_layernorm_gradients(gpu_lib, dtype, rows, n, pad, offset):
    t, tag, wt, u, half = kinds(dtype)
    x, g = laid(inputs.normal(55, (rows, n)) * 2.0 + 0.5, t, pad, offset), laid(inputs.normal(56, (rows, n)), t, pad, offset)
    gamma = vector(1.0 + 0.3 * inputs.normal(57, (n,)), t)
    xs = wide64(x)
    _, m, i = ref.layernorm_forward(xs, None, None, 1e-5)
    mean, inv = vector(m, wt), vector(i, wt)
    gi, gg, gb = room((rows, n), t, pad, offset), room((n,), wt), room((n,), wt)

    def call(grad_in, weights=True, gam=gamma.data_ptr()):
        eb.layernorm_gradients_device(g.data_ptr(), x.data_ptr(), mean.data_ptr(), inv.data_ptr(), gam, grad_in.data_ptr(),
                                      gg.data_ptr() if weights else 0, gb.data_ptr() if weights else 0, rows, n, tag,
                                      ld_grad_out=g.stride(0), ldx=x.stride(0), ld_grad_in=grad_in.stride(0))
        done()

    call(gi)
    gs, ws, ms, rs = wide64(g), wide64(gamma), wide64(mean), wide64(inv)
    want, wg, wb = ref.layernorm_gradients(gs, xs, ms, rs, ws)
    xhat, up = np.abs((xs - ms[:, None]) * rs[:, None]), np.abs(gs * ws)
    scale = rs[:, None] * (up.max(axis=1, keepdims=True) + up.mean(axis=1, keepdims=True)
                           + xhat.max(axis=1, keepdims=True) * (up * xhat).mean(axis=1, keepdims=True))
    assert np.all(np.abs(wide64(gi) - want) <= half * np.abs(want) + 200 * u * scale)
    # a group adds its rows one by one and the groups' shares are joined: fewer than 400 additions in a row
    assert np.all(np.abs(wide64(gg) - wg) <= 400 * u * (np.abs(gs) * xhat).sum(axis=0))
    assert np.all(np.abs(wide64(gb) - wb) <= 400 * u * np.abs(gs).sum(axis=0))
    assert untouched(gi, offset)
    first = (wide64(gi), wide64(gg), wide64(gb))
    call(gi)
    assert all(np.array_equal(a, b) for a, b in zip(first, (wide64(gi), wide64(gg), wide64(gb))))  # no order left to chance
    gg.fill_(3.0)
    import torch
    torch.cuda.synchronize()
    call(g, weights=False)  # in place of grad_out
    assert np.array_equal(wide64(g), first[0]) and bool((gg == 3.0).all())


VOCABS = [(1, 1, 0, 0), (3, 5, 0, 0), (70, 33, 7, 3), (5, 1000, 0, 0), (9, 2049, 1, 1), (300, 4097, 0, 0), (4, 50257, 0, 0),
          (2, 131072, 8, 8), (1, 200003, 0, 0), (700, 200, 0, 0)]


def logits(seed, rows, vocab, coarse=False):
    x = 3.0 * inputs.normal(seed, (rows, vocab))
    return np.round(x) if coarse else x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,pad,offset", VOCABS)
@pytest.mark.parametrize("how", ["plain", "ties", "masked", "equal"])
def test_token_logprobs(gpu_lib, dtype, rows, vocab, pad, offset, how):
    t, tag, wt, u, half = kinds(dtype)
    v = logits(61, rows, vocab, coarse=how == "ties")
    if how == "equal":  # more ties than there is room for candidates: the lowest indices win
        v[:] = 0.5
        v[0, vocab // 3:] = 0.25
    if how == "masked":
        v[inputs.uniform(62, (rows, vocab)) < 0.2] = -np.inf
        v[0, :] = -np.inf
        if rows > 2:
            v[2, :] = -np.inf
            v[2, vocab // 2] = -3.0
    x = laid(v, t, pad, offset)
    import torch
    tokens_np = (np.arange(rows) * 7919) % vocab
    tokens_np[4::5] = -1
    tokens = torch.from_numpy(tokens_np).cuda()
    k = min(vocab, [1, 8, 20, 32][rows % 4])
    lp, ent, lse = room((rows,), wt), room((rows,), wt), room((rows,), wt)
    tl, ti = room((rows, k), wt), torch.full((rows, k), -7, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    eb.token_logprobs_device(x.data_ptr(), tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), tl.data_ptr(),
                             ti.data_ptr(), rows, vocab, k, tag, ld=x.stride(0))
    done()
    xs = wide64(x)
    w_lp, w_ent, w_lse, w_tl, w_ti = ref.token_logprobs(xs, tokens_np, k)
    assert np.array_equal(ti.cpu().numpy(), w_ti)
    # a term exp(d) is off by (8 + 3 |d|) u of itself, the sum by 200 u more; |d| averages below 16
    s = 300 * u

    def close(got, want, tol):
        got = wide64(got)
        fin = np.isfinite(want)
        assert np.array_equal(got[~fin], want[~fin], equal_nan=True)
        assert np.all(np.abs(got[fin] - want[fin]) <= tol[fin])

    with np.errstate(invalid="ignore"):
        m = np.where(np.isfinite(w_lse), xs.max(axis=1), 0.0)
    close(lse, w_lse, s + 2 * u * np.abs(np.where(np.isfinite(w_lse), w_lse, 0)))
    span = np.where(np.isfinite(w_lse), np.abs(w_lse - m), 0)
    close(lp, w_lp, s + 4 * u * (np.abs(np.where(np.isfinite(w_lp), w_lp, 0)) + span))
    close(tl, w_tl, s + 4 * u * (np.abs(np.where(np.isfinite(w_tl), w_tl, 0)) + span[:, None]))
    close(ent, w_ent, 2 * s * (2.0 + np.log(vocab)) * np.ones(rows))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [700, 5000, 40000])
def test_token_logprobs_far_from_zero(gpu_lib, dtype, vocab):
    """Rows around a large level, as additive masks leave them: differences from the largest logit decide."""
    import torch
    t, tag, wt, u, half = kinds(dtype)
    levels = [0.0, 60.0, -70.0, 300.0, -5000.0, 60000.0] + ([] if dtype == "f16" else [1e6, -1e9, 1e12, -1e30, 1e35])
    rows = len(levels)
    x = laid(np.array(levels)[:, None] + inputs.normal(63, (rows, vocab)), t)
    tokens = torch.arange(rows, device="cuda") * 7
    lp, ent, lse = room((rows,), wt), room((rows,), wt), room((rows,), wt)
    eb.token_logprobs_device(x.data_ptr(), tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), 0, 0, rows,
                             vocab, 0, tag)
    done()
    xs = wide64(x)
    y = xs - xs.max(axis=1, keepdims=True)  # the same probabilities, and logprob without cancellation
    w_lp, w_ent, w_norm, _, _ = ref.token_logprobs(y, tokens.cpu().numpy(), 1)
    s = 300 * u  # as above
    w_lse = xs.max(axis=1) + w_norm
    assert np.all(np.abs(wide64(lse) - w_lse) <= s + 2 * u * np.abs(w_lse))
    assert np.all(np.abs(wide64(lp) - w_lp) <= s + 4 * u * (np.abs(w_lp) + w_norm))
    assert np.all(np.abs(wide64(ent) - w_ent) <= 2 * s * (2.0 + np.log(vocab)))


def test_token_logprobs_outputs_are_optional(gpu_lib):
    import torch
    t, tag, wt, u, half = kinds("bf16")
    x = laid(logits(63, 40, 3001), t)
    tokens = torch.arange(40, device="cuda")
    full = [room((40,), wt) for _ in range(3)]
    eb.token_logprobs_device(x.data_ptr(), tokens.data_ptr(), *[f.data_ptr() for f in full], 0, 0, 40, 3001, 0, tag)
    done()
    ti = torch.empty(40, 5, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    eb.token_logprobs_device(x.data_ptr(), 0, 0, 0, 0, 0, ti.data_ptr(), 40, 3001, 5, tag)
    done()
    assert np.array_equal(ti.cpu().numpy(), ref.token_logprobs(wide64(x), np.zeros(40, dtype=int), 5)[4])
    one = room((40,), wt)
    eb.token_logprobs_device(x.data_ptr(), 0, 0, one.data_ptr(), 0, 0, 0, 40, 3001, 0, tag)
    done()
    assert np.array_equal(wide64(one), wide64(full[1]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_of_rows_with_nan_infinity_and_lowest_values(gpu_lib, dtype):
    import torch
    t, tag, wt, u, half = kinds(dtype)
    low = torch.finfo(t).min
    v = logits(64, 6, 700)
    v[0, 5] = np.nan
    v[1, 9] = np.inf
    v[2, :] = np.nan
    v[2, 17] = 1.0
    v[3, :] = low          # nothing but the type's lowest value: a uniform row
    v[4, ::2] = low
    v[5, :] = -np.inf
    v[5, 100:] = low
    x = laid(v, t)
    tokens_np = np.array([0, 9, 17, 699, 1, 650])
    tokens = torch.from_numpy(tokens_np).cuda()
    lp, ent, lse = room((6,), wt), room((6,), wt), room((6,), wt)
    tl, ti = room((6, 8), wt), torch.empty(6, 8, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    eb.token_logprobs_device(x.data_ptr(), tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), tl.data_ptr(),
                             ti.data_ptr(), 6, 700, 8, tag)
    done()
    w_lp, w_ent, w_lse, w_tl, w_ti = ref.token_logprobs(wide64(x), tokens_np, 8)
    assert np.array_equal(ti.cpu().numpy(), w_ti)
    # rows 3 and 5 hold equal logits of the type's largest magnitude: the definition's difference x - lse
    # loses them in 64 bits, so they are compared by hand below
    for got, want in ((lp, w_lp), (ent, w_ent), (lse, w_lse), (tl, w_tl)):
        got, want = (np.delete(a, [3, 5], axis=0) for a in (wide64(got), want))
        fin = np.isfinite(want)
        assert np.array_equal(got[~fin], want[~fin], equal_nan=True)
        assert np.all(np.abs(got - want)[fin] <= 300 * u * (2 + np.abs(want[fin]) + np.log(700)))
    # the uniform rows, by hand
    for r, count in ((3, 700), (5, 600)):
        assert abs(wide64(ent)[r] - np.log(count)) <= 300 * u * 10
        assert abs(wide64(lp)[r] + np.log(count)) <= 300 * u * 10


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,pad,offset", VOCABS)
def test_token_logprobs_gradient(gpu_lib, dtype, rows, vocab, pad, offset):
    import torch
    t, tag, wt, u, half = kinds(dtype)
    v = logits(65, rows, vocab)
    v[inputs.uniform(66, (rows, vocab)) < 0.1] = -np.inf
    v[:, 0] = 1.0
    if rows > 1:
        v[1, :] = -np.inf
    x = laid(v, t, pad, offset)
    tokens_np = (np.arange(rows) * 31) % vocab
    tokens_np[2::4] = -1
    tokens = torch.from_numpy(tokens_np).cuda()
    xs = wide64(x)
    _, e, l = ref.token_logprobs(xs, tokens_np, 0)[:3]
    lse, ent = vector(l, wt), vector(e, wt)
    g, h = vector(inputs.normal(67, (rows,)), wt), vector(inputs.normal(68, (rows,)), wt)

    def check(gout, hout, out):
        gs = wide64(g) if gout else np.zeros(rows)
        hs = wide64(h) if hout else np.zeros(rows)
        ls, es = wide64(lse), wide64(ent)
        want = ref.token_logprobs_gradient(xs, tokens_np, ls, es, gs, hs)
        with np.errstate(all="ignore"):
            lpv = np.where(xs > -np.inf, xs - ls[:, None], 0.0)
            p = np.where(xs > -np.inf, np.exp(lpv), 0.0)
        mag = p * (np.abs(gs)[:, None] + np.abs(hs)[:, None] * (np.abs(lpv) + np.abs(es)[:, None]))
        # exp is off by (8 + 3 |lp|) u, the products by a few u; the storage type's smallest step, and
        # exponentials below 2^-126, which are zero
        tol = half * np.abs(want) + (16 + 8 * np.abs(lpv)) * u * mag + 2 * u * np.abs(gs)[:, None]
        tol = tol + torch.finfo(t).smallest_normal * torch.finfo(t).eps + (0 if dtype == "f64" else 2.0 ** -126 * 200)
        assert np.all(np.abs(wide64(out) - want) <= tol)

    out = room((rows, vocab), t, pad, offset)
    call = lambda o, gp, hp: (eb.token_logprobs_gradient_device(  # noqa: E731
        x.data_ptr(), tokens.data_ptr() if gp else 0, lse.data_ptr(), ent.data_ptr() if hp else 0, g.data_ptr() if gp else 0,
        h.data_ptr() if hp else 0, o.data_ptr(), rows, vocab, tag, ld=x.stride(0), ld_grad=o.stride(0)), done())
    call(out, True, True)
    check(True, True, out)
    assert untouched(out, offset)
    both = wide64(out)
    out.fill_(float("nan"))
    torch.cuda.synchronize()
    call(out, True, False)
    check(True, False, out)
    call(out, False, True)
    check(False, True, out)
    # another alignment of the result than of the logits
    other = room((rows, vocab), t, pad + 1, 1)
    call(other, True, True)
    assert np.array_equal(wide64(other), both)
    # in place
    if pad == 0:
        call(x, True, True)
        assert np.array_equal(wide64(x), both)


def test_tokens_outside_the_vocabulary_make_their_row_nan(gpu_lib):
    import torch
    t, tag, wt, u, half = kinds("f32")
    x = laid(logits(69, 3, 100), t)
    tokens = torch.tensor([5, 100, 1 << 40], device="cuda")
    lp, ent, lse, g = (room((3,), wt) for _ in range(4))
    g.fill_(1.0)
    torch.cuda.synchronize()
    eb.token_logprobs_device(x.data_ptr(), tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), 0, 0, 3, 100, 0, tag)
    out = room((3, 100), t)
    eb.token_logprobs_gradient_device(x.data_ptr(), tokens.data_ptr(), lse.data_ptr(), 0, g.data_ptr(), 0, out.data_ptr(), 3, 100, tag)
    done()
    assert np.isnan(wide64(lp)[1:]).all() and np.isfinite(wide64(lp)[0]) and np.isfinite(wide64(lse)).all()
    assert np.isnan(wide64(out)[1:]).all() and np.isfinite(wide64(out)[0]).all()


def test_refusals_and_empty_calls(gpu_lib):
    import torch
    lib = gpu_lib
    x = room((4, 8), torch.float32, fill=1.0)
    v = room((8,), torch.float32, fill=7.0)
    p, o = x.data_ptr(), v.data_ptr()
    q = room((4, 8), torch.float32).data_ptr()
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    F32 = eb.DTYPE_F32
    norm, grads = lib.eshkol_b200_layernorm_forward_device, lib.eshkol_b200_layernorm_gradients_device
    assert norm(p, o, o, q, None, None, 4, 0, 0, 0, 1e-5, F32) == -1       # no features
    assert norm(p, o, o, q, None, None, 4, 8, 7, 0, 1e-5, F32) == -1       # pitch shorter than a row
    assert norm(p, o, o, q, None, None, 4, 8, 0, 0, -1.0, F32) == -1       # epsilon
    assert norm(p, o, o, q, None, None, 4, 8, 0, 0, float("nan"), F32) == -1
    assert norm(p, o, o, q, None, None, 4, 8, 0, 0, 1e-5, 4) == -1         # no such type
    assert norm(p, o, o, p, None, None, 4, 8, 8, 9, 1e-5, F32) == -1       # in place with another pitch
    assert norm(None, o, o, q, None, None, 4, 8, 0, 0, 1e-5, F32) == -1
    assert norm(None, None, None, None, None, None, 0, 8, 0, 0, 1e-5, F32) == 0  # no samples
    assert grads(p, p, o, o, None, p, None, None, 4, 8, 8, 8, 9, F32) == -1
    assert grads(p, q, o, o, None, q, None, None, 4, 8, 0, 0, 0, F32) == -1      # grad_in over x
    assert grads(p, q, None, o, None, p, None, None, 4, 8, 0, 0, 0, F32) == -1   # no statistics
    logp, glog = lib.eshkol_b200_token_logprobs_device, lib.eshkol_b200_token_logprobs_gradient_device
    t, q2 = tok.data_ptr(), v.data_ptr()
    assert logp(p, None, q2, None, None, None, None, 4, 8, 0, 0, F32) == -1      # logprob without tokens
    assert logp(p, t, None, None, None, None, None, 4, 8, 0, 0, F32) == -1       # nothing asked for
    assert logp(p, t, q2, None, None, None, None, 4, 8, 0, 3, F32) == -1         # alternatives without a place
    assert logp(p, t, q2, None, None, q, None, 4, 8, 0, 0, F32) == -1            # a place without alternatives
    assert logp(p, t, q2, None, None, q, None, 4, 8, 0, 9, F32) == -1            # more than the vocabulary
    assert logp(p, t, q2, None, None, q, None, 4, 800, 0, 33, F32) == -1         # more than 32
    assert logp(p, t, q2, None, None, None, None, 4, 8, 7, 0, F32) == -1
    assert logp(p, t, q2, None, None, None, None, 4, 0, 0, 0, F32) == -1
    assert logp(None, None, None, q2, None, None, None, 0, 8, 0, 0, F32) == 0
    assert glog(p, None, q2, None, q2, None, q, 4, 8, 0, 0, F32) == -1           # tokens missing
    assert glog(p, t, q2, None, None, q2, q, 4, 8, 0, 0, F32) == -1              # entropy missing
    assert glog(p, t, q2, q2, None, None, q, 4, 8, 0, 0, F32) == -1              # no gradient at all
    assert glog(p, t, q2, None, q2, None, p, 4, 8, 8, 9, F32) == -1
    assert glog(None, t, q2, None, q2, None, None, 0, 8, 0, 0, F32) == 0
    # sums over no samples
    assert grads(None, None, None, None, None, None, o, None, 0, 8, 0, 0, 0, F32) == 0
    done()
    assert bool((v == 0).all())


def test_captured_calls_own_their_scratch(gpu_lib):
    """Two graphs captured from the library's stream and an eager call of a larger size between their
    replays: nobody's scratch is anybody else's."""
    import torch
    t, tag, wt, u, half = kinds("bf16")
    stream = torch.cuda.ExternalStream(api.stream_handle())

    def case(seed, rows, n):
        x, g = laid(inputs.normal(seed, (rows, n)), t), laid(inputs.normal(seed + 1, (rows, n)), t)
        _, m, i = ref.layernorm_forward(wide64(x), None, None, 1e-5)
        s = dict(x=x, g=g, mean=vector(m, wt), inv=vector(i, wt), gi=room((rows, n), t), gg=room((n,), wt), gb=room((n,), wt))
        s["call"] = lambda: eb.layernorm_gradients_device(  # noqa: E731
            g.data_ptr(), x.data_ptr(), s["mean"].data_ptr(), s["inv"].data_ptr(), 0, s["gi"].data_ptr(), s["gg"].data_ptr(),
            s["gb"].data_ptr(), rows, n, tag)
        return s

    a, b, big = case(71, 300, 512), case(73, 500, 1000), case(75, 2000, 4096)
    want = []
    for s in (a, b):
        s["call"]()
        done()
        want.append((wide64(s["gi"]), wide64(s["gg"]), wide64(s["gb"])))
        for k in ("gi", "gg", "gb"):
            s[k].fill_(float("nan"))
    torch.cuda.synchronize()
    graphs = []
    for s in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s["call"]()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(stream):
            graphs[1].replay()
        big["call"]()
    torch.cuda.synchronize()
    done()
    for s, w in zip((a, b), want):
        assert all(np.array_equal(x, wide64(s[k])) for x, k in zip(w, ("gi", "gg", "gb")))
