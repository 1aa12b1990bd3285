"""The logits' gradient where nothing is left of a row or its factors are large."""
import numpy as np
import pytest

import eshkol_b200 as eb
from oracle import operators_ref as ref
from test_gpu_norm_logprobs import done, kinds, laid, logits, room, vector, wide64

pytestmark = pytest.mark.gpu


def gradient(x, tokens, lse, ent, g, h, tag, wt):
    import torch
    rows, vocab = x.shape
    tok = torch.from_numpy(np.asarray(tokens)).cuda()
    ls, es, gs, hs = (vector(np.asarray(v, dtype=np.float64), wt) for v in (lse, ent, g, h))
    out = room((rows, vocab), x.dtype)
    eb.token_logprobs_gradient_device(x.data_ptr(), tok.data_ptr(), ls.data_ptr(), es.data_ptr(), gs.data_ptr(), hs.data_ptr(),
                                      out.data_ptr(), rows, vocab, tag, ld=x.stride(0))
    done()
    return wide64(out), [wide64(v) for v in (ls, es, gs, hs)]


@pytest.mark.parametrize("dtype", ["f64", "f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [5, 700, 9001])
def test_a_large_gradient_of_the_entropy_meets_masked_entries(gpu_lib, dtype, vocab):
    """Masked entries stay at zero and the others at their values, however large the factor in front of
    p log p is (a scaled loss, say)."""
    t, tag, wt, u, half = kinds(dtype)
    v = logits(141, 4, vocab)
    v[:, 1::3] = -np.inf
    x = laid(v, t)
    xs = wide64(x)
    tokens = np.array([0, 2, -1, 3])
    _, ent, lse = ref.token_logprobs(xs, tokens, 0)[:3]
    scale = 1e3 if dtype == "f16" else 1e12  # f16 results would be infinite beyond
    g, h = np.array([1.0, -2.0, 3.0, 0.0]), scale * np.array([1.0, -1.0, 4.0, 2.5])
    got, (ls, es, gs, hs) = gradient(x, tokens, lse, ent, g, h, tag, wt)
    want = ref.token_logprobs_gradient(xs, tokens, ls, es, gs, hs)
    assert np.isfinite(want).all()
    assert (got[np.isneginf(xs)] == 0.0).all()
    with np.errstate(all="ignore"):
        lp = np.where(xs > -np.inf, xs - ls[:, None], 0.0)
        p = np.where(xs > -np.inf, np.exp(lp), 0.0)
    # as in the sweep over shapes: exp is off by (8 + 3 |lp|) u, the products by a few u
    mag = p * (np.abs(gs)[:, None] + np.abs(hs)[:, None] * (np.abs(lp) + np.abs(es)[:, None]))
    tol = half * np.abs(want) + (16 + 8 * np.abs(lp)) * u * mag + 2 * u * np.abs(gs)[:, None] + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert np.all(np.abs(got - want) <= tol + (0 if dtype == "f64" else 2.0 ** -126 * 200 * np.abs(hs)[:, None]))


@pytest.mark.parametrize("dtype", ["f64", "f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 7, 900, 20001])
def test_a_row_without_unmasked_entries(gpu_lib, dtype, vocab):
    """All its probabilities are zero: what is left of the formula is grad_logprob at the token, and zeros."""
    t, tag, wt, u, half = kinds(dtype)
    x = laid(np.full((4, vocab), -np.inf), t)
    tokens = np.array([0, vocab // 2, -1, vocab - 1])
    nothing = np.full(4, -np.inf)
    g, h = np.array([2.0, -0.5, 3.0, 0.0]), np.array([1.0, -4.0, 2.0, 0.25])
    got, _ = gradient(x, tokens, nothing, np.zeros(4), g, h, tag, wt)
    want = np.zeros((4, vocab))
    want[0, 0], want[1, vocab // 2] = 2.0, -0.5
    assert np.array_equal(got, want)
    # the forward pass gives the lse and entropy used here
    import torch
    lp, ent, lse = (room((4,), wt) for _ in range(3))
    tok = torch.from_numpy(tokens).cuda()
    torch.cuda.synchronize()
    eb.token_logprobs_device(x.data_ptr(), tok.data_ptr(), lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), 0, 0, 4, vocab, 0, tag)
    done()
    assert np.array_equal(wide64(lse), nothing) and np.array_equal(wide64(ent), np.zeros(4))
    assert np.array_equal(wide64(lp), [-np.inf, -np.inf, 0.0, -np.inf])
