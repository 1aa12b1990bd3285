"""CPU restatement (test infrastructure, not part of the product) of the reference's tensor
operators beside the matrix product, lib/backend/gpu/gpu_cuda_kernels.cu: reduce :76-141 and its
CPU twin lib/backend/gpu/gpu_memory_cuda.cpp:1247-1268, axis reduce :147-180, transpose :189-213,
softmax :319-343, normalize :364-389, batchnorm backward :489-521, layernorm backward :524-555.

numpy sums are pairwise where the reference's loops are serial, and the GPU kernels under test
share each sum between threads: the three agree to rounding, which is what the tests assert.
"""
import numpy as np

SUM, PROD, MIN, MAX, MEAN = range(5)


def reduce_all(x, op):
    x = np.asarray(x, dtype=np.float64).ravel()
    if op == SUM:
        return float(np.sum(x))
    if op == PROD:
        return float(np.prod(x))
    if op == MIN:
        return float(np.fmin.reduce(x, initial=np.inf))   # fmin / fmax: a NaN operand is ignored
    if op == MAX:
        return float(np.fmax.reduce(x, initial=-np.inf))
    if op == MEAN:
        return float(np.sum(x) / x.size)
    raise ValueError(op)


def reduce_axis(x, axis, op):
    x = np.asarray(x, dtype=np.float64)
    if op == SUM:
        return np.sum(x, axis=axis)
    if op == PROD:
        return np.prod(x, axis=axis)
    if op == MIN:
        return np.fmin.reduce(x, axis=axis, initial=np.inf)
    if op == MAX:
        return np.fmax.reduce(x, axis=axis, initial=-np.inf)
    if op == MEAN:
        return np.sum(x, axis=axis) / x.shape[axis]
    raise ValueError(op)


def softmax(x):
    """x: [slices, len]; the maximum is subtracted first and a zero sum divides by 1."""
    x = np.asarray(x, dtype=np.float64)
    m = np.fmax.reduce(x, axis=1, keepdims=True)
    e = np.exp(x - m)
    s = e.sum(axis=1, keepdims=True)
    s[s == 0.0] = 1.0
    return e / s


def normalize(x, gamma, beta, eps):
    """x: [slices, len]; scalar gamma / beta, population variance."""
    x = np.asarray(x, dtype=np.float64)
    n = x.shape[1]
    mean = x.sum(axis=1, keepdims=True) / n
    var = ((x - mean) ** 2).sum(axis=1, keepdims=True) / n
    return gamma * (x - mean) * (1.0 / np.sqrt(var + eps)) + beta


def batchnorm_backward(grad_out, x, mean, inv_std, gamma):
    """grad_out, x: [batch, features]; mean, inv_std, gamma: [features].
    Returns grad_input, grad_gamma, grad_beta."""
    N = grad_out.shape[0]
    nz = (x - mean) * inv_std
    sum_g = grad_out.sum(axis=0)
    sum_gn = (grad_out * nz).sum(axis=0)
    coeff = gamma * inv_std / N
    return coeff * (N * grad_out - sum_g - nz * sum_gn), sum_gn, sum_g


def layernorm_backward(grad_out, x, mean, inv_std, gamma):
    """grad_out, x: [samples, features]; mean, inv_std: [samples]; gamma: [features]."""
    D = grad_out.shape[1]
    g = grad_out * gamma
    nz = (x - mean[:, None]) * inv_std[:, None]
    sum_g = g.sum(axis=1, keepdims=True)
    sum_gn = (g * nz).sum(axis=1, keepdims=True)
    return (inv_std[:, None] / D) * (D * g - sum_g - nz * sum_gn)


# ---- training and serving operators, in f64 from their definitions (no counterpart in the reference)
def layernorm_forward(x, gamma, beta, eps):
    """(y, mean, inv_std) of layer normalisation with weight vectors."""
    x = np.asarray(x, dtype=np.float64)
    mean = x.mean(axis=1)
    inv_std = 1.0 / np.sqrt(((x - mean[:, None]) ** 2).mean(axis=1) + eps)
    y = (x - mean[:, None]) * inv_std[:, None]
    return y * (1.0 if gamma is None else gamma) + (0.0 if beta is None else beta), mean, inv_std


def layernorm_gradients(g, x, mean, inv_std, gamma):
    """(grad_in, grad_gamma, grad_beta) from saved statistics."""
    xhat = (x - mean[:, None]) * inv_std[:, None]
    u = g * (1.0 if gamma is None else gamma)
    n = x.shape[1]
    grad_in = inv_std[:, None] * (u - u.sum(axis=1, keepdims=True) / n - xhat * (u * xhat).sum(axis=1, keepdims=True) / n)
    return grad_in, (g * xhat).sum(axis=0), g.sum(axis=0)


def token_logprobs(x, tokens, n_top):
    """(logprob, entropy, lse, top_logprob, top_index): masked entries are minus infinity, a negative
    token stands for none, equal logits go by index.  A row with NaN or plus infinity is NaN and its
    alternatives are those of its numbers (index -1 where there are too few)."""
    x = np.asarray(x, dtype=np.float64)
    rows, vocab = x.shape
    bad = (np.isnan(x) | (x == np.inf)).any(axis=1)
    with np.errstate(all="ignore"):
        m = np.where(np.isnan(x), -np.inf, x).max(axis=1)
        m0 = np.where(np.isfinite(m), m, 0.0)[:, None]
        e = np.where(np.isnan(x), 0.0, np.exp(np.where(x == np.inf, 0.0, x - m0)))
        s = e.sum(axis=1)
        lse = np.where(bad, np.nan, m0[:, 0] + np.log(s))
        d = np.where(e > 0, x - m0, 0.0)
        ent = np.where(bad, np.nan, np.where(s > 0, np.log(s) - (e * d).sum(axis=1) / np.where(s > 0, s, 1.0), 0.0))

        def log_prob(v, l):
            return np.where(np.isnan(l), np.nan, np.where(v == -np.inf, -np.inf, v - l))

        logprob = np.zeros(rows)
        for r in range(rows):
            if tokens[r] >= vocab:
                logprob[r] = np.nan
            elif tokens[r] >= 0:
                logprob[r] = log_prob(x[r, tokens[r]], lse[r])
        top_lp, top_i = np.full((rows, n_top), np.nan), np.full((rows, n_top), -1, dtype=np.int64)
        for r in range(rows):
            order = np.argsort(np.where(np.isnan(x[r]), np.inf, -x[r]), kind="stable")
            order = order[~np.isnan(x[r][order])][:n_top]
            top_i[r, :len(order)] = order
            top_lp[r, :len(order)] = log_prob(x[r][order], lse[r])
    return logprob, ent, lse, top_lp, top_i


def token_logprobs_gradient(x, tokens, lse, entropy, g, h):
    """Gradient of the logits; g, h: gradients of logprob and entropy."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(all="ignore"):
        lp = x - lse[:, None]
        p = np.where(lse[:, None] == -np.inf, 0.0, np.exp(lp))
        g = np.where(tokens >= 0, g, 0.0)
        grad = -p * g[:, None] - h[:, None] * np.where(p > 0, p * (lp + entropy[:, None]), 0.0)
    for r in range(x.shape[0]):
        if tokens[r] >= x.shape[1]:
            grad[r] = np.nan
        elif tokens[r] >= 0:
            grad[r, tokens[r]] += g[r]
    return grad


GELU_A, GELU_B = np.sqrt(2.0 / np.pi), 0.044715


def activate(z, act):
    """0 none, 1 ReLU, 2 the tanh form of GELU."""
    if act == 1:
        return np.where(z > 0, z, 0.0)
    if act == 2:
        return 0.5 * z * (1.0 + np.tanh(GELU_A * (z + GELU_B * z ** 3)))
    return z


def activate_slope(z, act):
    if act == 1:
        return (z > 0).astype(np.float64)
    if act == 2:
        t = np.tanh(GELU_A * (z + GELU_B * z ** 3))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_A * (1.0 + 3.0 * GELU_B * z ** 2)
    return np.ones_like(z)


def linear_forward(x, w, bias, residual, act):
    """(y, pre) of the linear layer, w [d_in x d_out]."""
    z = x @ w + (0.0 if bias is None else bias)
    return activate(z, act) + (0.0 if residual is None else residual), z


def linear_gradients(g, x, w, pre, act):
    """(grad_x, grad_w, grad_bias, dz)."""
    dz = g * activate_slope(pre, act) if act else g
    return dz @ w.T, x.T @ dz, dz.sum(axis=0), dz


# ---- f32 products by bf16 parts, as the linear layer multiplies them
def to_bf16(x):
    """f32 values rounded to the nearest bf16 (ties to even), as f32; finite input"""
    b = np.asarray(x, dtype=np.float32).view(np.uint32)
    b = (b + np.uint32(0x7FFF) + ((b >> np.uint32(16)) & np.uint32(1))) & np.uint32(0xFFFF0000)
    return b.view(np.float32)


def bf16_parts(x, count=3):
    """The leading `count` parts of f32 values; three of them add up to the value."""
    rest, parts = np.asarray(x, dtype=np.float32), []
    for _ in range(count):
        parts.append(to_bf16(rest))
        rest = (rest - parts[-1]).astype(np.float32)
    return parts


def product_of_parts(x, w, count=3):
    """x @ w in f64 from the products of parts i, j with i + j < count (six of nine for three parts)"""
    a, b = ([p.astype(np.float64) for p in bf16_parts(v, count)] for v in (x, w))
    return sum(a[i] @ b[j] for i in range(count) for j in range(count - i))
