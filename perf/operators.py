"""Cases of the training and serving operators on device tensors: layer normalisation with affine weights
and its three gradients, the linear layer with bias, activation and residual and its gradients, and the
log probabilities of given tokens with entropy and top alternatives and their gradient.

With `own` false `run` computes each operator in plain torch operations (32 bits, 64 for f64 tensors),
with `own` true it calls the library.  Sizes: feature and hidden widths as dense language models have
them, vocabularies from tens of thousands to over a hundred thousand entries (odd ones included, so
rows start off any 16-byte boundary), token counts from one decoded token to a packed training batch.
"""
import math

import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
ACT = {"none": 0, "relu": 1, "gelu": 2}
EPS = 1e-5
GELU_A, GELU_B = math.sqrt(2.0 / math.pi), 0.044715


def listed():
    return [
        # the norm before a block while one token is decoded: nothing but latency
        {"name": "norm token", "op": "norm", "dtype": "bf16", "rows": 1, "features": 4096, "pad": 0, "offset": 0},
        # the norm over a batch of prompts, statistics kept for the backward pass
        {"name": "norm prompt", "op": "norm", "dtype": "bf16", "rows": 8192, "features": 4096, "pad": 0, "offset": 0},
        # its gradients in a training step, weight gradients reduced over the tokens of the batch
        {"name": "norm gradients", "op": "norm_grad", "dtype": "bf16", "rows": 16384, "features": 4096, "pad": 0, "offset": 0},
        # f64 tensors, as programs of this framework hold them: odd width, rows of a wider buffer
        {"name": "norm gradients f64", "op": "norm_grad", "dtype": "f64", "rows": 1537, "features": 1001, "pad": 6, "offset": 1},
        # the up projection while one token is decoded: the weights are read once
        {"name": "linear token", "op": "linear", "dtype": "bf16", "rows": 1, "d_in": 4096, "d_out": 16384, "act": "gelu",
         "bias": True, "residual": False, "pre": False, "trans_w": False, "pad": 0, "offset": 0},
        # the down projection of a batch of prompts, added to the residual stream
        {"name": "linear prompt", "op": "linear", "dtype": "bf16", "rows": 8192, "d_in": 16384, "d_out": 4096, "act": "none",
         "bias": True, "residual": True, "pre": False, "trans_w": False, "pad": 0, "offset": 0},
        # f32 weights, ragged sizes, rows that start on no 16-byte boundary
        {"name": "linear f32 ragged", "op": "linear", "dtype": "f32", "rows": 777, "d_in": 2001, "d_out": 1603, "act": "gelu",
         "bias": True, "residual": True, "pre": True, "trans_w": False, "pad": 3, "offset": 1},
        # all gradients of the up projection in a training step
        {"name": "linear gradients", "op": "linear_grad", "dtype": "bf16", "rows": 4096, "d_in": 4096, "d_out": 16384, "act": "gelu",
         "bias": True, "trans_w": False, "pad": 0, "offset": 0},
        # a small layer of odd sizes, weights stored output by input
        {"name": "linear gradients ragged", "op": "linear_grad", "dtype": "f16", "rows": 333, "d_in": 1001, "d_out": 1999, "act": "relu",
         "bias": True, "trans_w": True, "pad": 5, "offset": 3},
        # scoring a batch of sequences: the given tokens, entropy and eight alternatives; odd vocabulary
        {"name": "logprobs prompt", "op": "logprobs", "dtype": "bf16", "rows": 4096, "vocab": 50257, "top": 8, "masked": False, "pad": 0, "offset": 0},
        # a few decoded tokens over a large vocabulary, part of it masked out
        {"name": "logprobs decode", "op": "logprobs", "dtype": "f32", "rows": 4, "vocab": 131072, "top": 20, "masked": True, "pad": 0, "offset": 0},
        # the loss's gradient with respect to the logits, with an entropy bonus
        {"name": "logprobs gradient", "op": "logprobs_grad", "dtype": "bf16", "rows": 4096, "vocab": 50257, "masked": False, "pad": 0, "offset": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "linear", "linear_grad", "logprobs", "logprobs_grad"])
    # half of the cases lie densely on aligned rows, the others are views of wider buffers
    pad, offset = (0, 0) if rng.random() < 0.5 else (rng.choice([3, 8, 17]), rng.choice([0, 1, 8]))
    offset = min(offset, pad)
    if op in ("norm", "norm_grad"):
        features = _log(rng, 16, 20000)
        rows = _log(rng, 1, min(30000, (1 << 25) // features))
        return {"op": op, "dtype": rng.choice(["f64", "f32", "f16", "bf16"]), "rows": rows, "features": features, "pad": pad, "offset": offset}
    if op in ("linear", "linear_grad"):
        dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
        d_in, d_out = _log(rng, 32, 8192), _log(rng, 32, 8192)
        if rng.random() < 0.5:
            d_in, d_out = (d_in + 31) // 32 * 32, (d_out + 31) // 32 * 32
        rows = _log(rng, 1, max(1, min(8192, (1 << 35) // (d_in * d_out))))
        case = {"op": op, "dtype": dtype, "rows": rows, "d_in": d_in, "d_out": d_out, "act": rng.choice(["none", "relu", "gelu"]),
                "bias": rng.random() < 0.7, "trans_w": rng.random() < 0.4, "pad": pad, "offset": offset}
        if op == "linear":
            case["residual"] = rng.random() < 0.5
            case["pre"] = rng.random() < 0.3
        return case
    vocab = _log(rng, 200, 160000)
    rows = _log(rng, 1, max(1, min(8192, (1 << 26) // vocab)))
    case = {"op": op, "dtype": rng.choice(["f64", "f32", "f16", "bf16"]), "rows": rows, "vocab": vocab, "masked": rng.random() < 0.4, "pad": pad, "offset": offset}
    if op == "logprobs":
        case["top"] = rng.choice([0, 1, 5, 20, 32])
    return case


def _stat(dtype):
    """The type of statistics and of vector gradients: f64 for f64 tensors, else f32."""
    return torch.float64 if dtype is torch.float64 else torch.float32


def _rows_of(rows, cols, pad, offset, dtype):
    """An uninitialised rows x cols view of a buffer with rows of cols + pad elements, `offset` of them in front."""
    return torch.empty(rows, cols + pad, dtype=dtype, device="cuda")[:, offset:offset + cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    wide = _stat(dtype)
    pad, offset, rows = case["pad"], case["offset"], case["rows"]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=wide) * scale + shift

    def laid(values):
        out = _rows_of(values.shape[0], values.shape[1], pad, offset, dtype)
        out.copy_(values)
        return out

    def room(r, c, t=dtype):
        return _rows_of(r, c, pad, offset, t)

    s = dict(case, torch_dtype=dtype)
    op = case["op"]
    if op in ("norm", "norm_grad"):
        n = case["features"]
        # a residual stream: a mean away from zero, rows of different size, a few large channels
        x = normal(rows, n) * torch.exp(0.5 * normal(rows, 1)) + 0.5 * normal(1, n)
        x[:, :: max(1, n // 7)] *= 8.0
        s["x"] = laid(x)
        s["gamma"], s["beta"] = normal(n, scale=0.2, shift=1.0).to(dtype), normal(n, scale=0.1).to(dtype)
        s["mean"], s["inv_std"] = torch.empty(rows, dtype=wide, device="cuda"), torch.empty(rows, dtype=wide, device="cuda")
        if op == "norm":
            s["y"] = room(rows, n)
        else:
            v = s["x"].to(wide)
            s["mean"].copy_(v.mean(dim=1))
            s["inv_std"].copy_(torch.rsqrt(v.var(dim=1, unbiased=False) + EPS))
            s["grad_out"], s["grad_in"] = laid(normal(rows, n)), room(rows, n)
            s["grad_gamma"], s["grad_beta"] = torch.empty(n, dtype=wide, device="cuda"), torch.empty(n, dtype=wide, device="cuda")
    elif op in ("linear", "linear_grad"):
        k, n = case["d_in"], case["d_out"]
        s["x"] = laid(normal(rows, k))
        s["w"] = laid(normal(*((n, k) if case["trans_w"] else (k, n)), scale=1.0 / math.sqrt(k)))
        s["bias"] = normal(n, scale=0.3).to(dtype) if case["bias"] else None
        if op == "linear":
            s["residual"] = laid(normal(rows, n)) if case["residual"] else None
            s["y"], s["z"] = room(rows, n), room(rows, n) if case["pre"] else None
        else:
            s["z"] = laid(normal(rows, n)) if case["act"] != "none" else None
            s["grad_out"] = laid(normal(rows, n))
            s["grad_x"], s["grad_w"] = room(rows, k), room(*s["w"].shape)
            s["grad_bias"] = torch.empty(n, dtype=wide, device="cuda") if case["bias"] else None
    else:
        v = case["vocab"]
        # logits with a few likely tokens in every row
        x = normal(rows, v, scale=2.0)
        at = torch.randint(v, (rows, 4), generator=gen, device="cuda")
        x.scatter_add_(1, at, 3.0 * normal(rows, 4).abs() + 2.0)
        if case["masked"]:  # a constrained vocabulary: a third of the entries are out
            x.masked_fill_(torch.rand(rows, v, generator=gen, device="cuda") < 1.0 / 3.0, -math.inf)
        s["logits"] = laid(x)
        del x
        # the sampled token is usually a likely one; every ninth position is padding (no token)
        tokens = at[:, 0].clone()
        tokens[::3] = torch.randint(v, (tokens[::3].numel(),), generator=gen, device="cuda")
        tokens[8::9] = -1
        s["tokens"] = tokens
        for name in ("logprob", "entropy", "lse"):
            s[name] = torch.empty(rows, dtype=wide, device="cuda")
        if op == "logprobs":
            s["top_logprob"] = torch.empty(rows, case["top"], dtype=wide, device="cuda")
            s["top_index"] = torch.empty(rows, case["top"], dtype=torch.int64, device="cuda")
        else:
            lse, ent = _lse_entropy(s["logits"].to(wide))
            s["lse"].copy_(lse)
            s["entropy"].copy_(ent)
            s["grad_logprob"], s["grad_entropy"] = normal(rows), normal(rows, scale=0.1)
            s["grad_logits"] = room(rows, v)
    return s


# ------------------------------------------------------------------ plain forms
def _lse_entropy(x):
    m = x.max(dim=1, keepdim=True).values
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(x - m)
    total = e.sum(dim=1, keepdim=True)
    # entropy = log(total) - sum e (x - m) / total; an entry of weight zero adds nothing
    part = torch.where(e > 0, e * (x - m), torch.zeros_like(e)).sum(dim=1, keepdim=True)
    ent = torch.where(total > 0, torch.log(total) - part / total, torch.zeros_like(total))
    return (m + torch.log(total))[:, 0], ent[:, 0]


def _act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(GELU_A * (z + GELU_B * z * z * z)))
    return z


def _act_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    t = torch.tanh(GELU_A * (z + GELU_B * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_A * (1.0 + 3.0 * GELU_B * z * z)


def _plain(s):
    dtype = s["torch_dtype"]
    wide = _stat(dtype)
    op = s["op"]
    if op == "norm":
        x = s["x"].to(wide)
        mean = x.mean(dim=1, keepdim=True)
        d = x - mean
        inv_std = 1.0 / torch.sqrt((d * d).mean(dim=1, keepdim=True) + EPS)
        y = d * inv_std * s["gamma"].to(wide) + s["beta"].to(wide)
        return {"y": y.to(dtype), "mean": mean[:, 0], "inv_std": inv_std[:, 0]}
    if op == "norm_grad":
        g = s["grad_out"].to(wide)
        inv_std = s["inv_std"][:, None]
        xhat = (s["x"].to(wide) - s["mean"][:, None]) * inv_std
        gw = g * s["gamma"].to(wide)
        grad_in = inv_std * (gw - gw.mean(dim=1, keepdim=True) - xhat * (gw * xhat).mean(dim=1, keepdim=True))
        return {"grad_in": grad_in.to(dtype), "grad_gamma": (g * xhat).sum(dim=0), "grad_beta": g.sum(dim=0)}
    if op == "linear":
        w = s["w"].to(wide)
        z = s["x"].to(wide) @ (w.t() if s["trans_w"] else w)
        if s["bias"] is not None:
            z = z + s["bias"].to(wide)
        y = _act(z, s["act"])
        if s["residual"] is not None:
            y = y + s["residual"].to(wide)
        return {"y": y.to(dtype), "pre": z.to(dtype) if s["pre"] else None}
    if op == "linear_grad":
        dz = s["grad_out"].to(wide)
        if s["z"] is not None:
            dz = dz * _act_slope(s["z"].to(wide), s["act"])
        w, x = s["w"].to(wide), s["x"].to(wide)
        grad_x = dz @ (w if s["trans_w"] else w.t())
        grad_w = dz.t() @ x if s["trans_w"] else x.t() @ dz
        return {"grad_x": grad_x.to(dtype), "grad_w": grad_w.to(dtype), "grad_bias": dz.sum(dim=0) if s["grad_bias"] is not None else None}
    x = s["logits"].to(wide)
    tokens = s["tokens"]
    given = tokens >= 0
    index = tokens.clamp(min=0)[:, None]
    none = torch.full((), -math.inf, dtype=wide, device=x.device)
    if op == "logprobs":
        lse, ent = _lse_entropy(x)
        picked = x.gather(1, index)[:, 0]
        logprob = torch.where(given, torch.where(picked == -math.inf, none, picked - lse), torch.zeros_like(lse))
        out = {"logprob": logprob, "entropy": ent, "lse": lse}
        if s["top"]:
            values, order = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
            values = values[:, :s["top"]]
            out["top_logprob"] = torch.where(values == -math.inf, none, values - lse[:, None])
            out["top_index"] = order[:, :s["top"]].contiguous()
        return out
    lp = x - s["lse"][:, None]
    p = torch.where(x == -math.inf, torch.zeros_like(x), torch.exp(lp))
    g = torch.where(given, s["grad_logprob"], torch.zeros_like(s["grad_logprob"]))[:, None]
    slope = torch.where(p > 0, p * (lp + s["entropy"][:, None]), torch.zeros_like(p))
    grad = -g * p - s["grad_entropy"][:, None] * slope
    grad.scatter_add_(1, index, g)
    return {"grad_logits": grad.to(dtype)}


# ------------------------------------------------------------------ the library's calls
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own(s):
    """The calls, on the library's stream, where the program's torch work moves with its first call: what torch has
    written comes before them, what it does with the results behind them."""
    import eshkol_b200 as eb

    if "moved" not in s:
        eb.load_library().eshkol_gpu_init()
        library = torch.cuda.ExternalStream(eb.stream_handle())
        library.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(library)
        s["moved"] = True
    return _calls(s, eb)


def _calls(s, eb):
    dtype = {torch.float64: eb.DTYPE_F64, torch.float32: eb.DTYPE_F32, torch.float16: eb.DTYPE_F16, torch.bfloat16: eb.DTYPE_BF16}[s["torch_dtype"]]
    op = s["op"]
    if op == "norm":
        x, y = s["x"], s["y"]
        eb.layernorm_device(x.data_ptr(), _ptr(s["gamma"]), _ptr(s["beta"]), y.data_ptr(), _ptr(s["mean"]), _ptr(s["inv_std"]),
                            s["rows"], s["features"], EPS, dtype, ldx=x.stride(0), ldy=y.stride(0))
        return {"y": y, "mean": s["mean"], "inv_std": s["inv_std"]}
    if op == "norm_grad":
        eb.layernorm_gradients_device(_ptr(s["grad_out"]), _ptr(s["x"]), _ptr(s["mean"]), _ptr(s["inv_std"]), _ptr(s["gamma"]),
                                      _ptr(s["grad_in"]), _ptr(s["grad_gamma"]), _ptr(s["grad_beta"]), s["rows"], s["features"], dtype,
                                      ld_grad_out=s["grad_out"].stride(0), ldx=s["x"].stride(0), ld_grad_in=s["grad_in"].stride(0))
        return {"grad_in": s["grad_in"], "grad_gamma": s["grad_gamma"], "grad_beta": s["grad_beta"]}
    if op == "linear":
        opts = eb.make_linear_opts(dtype, activation=ACT[s["act"]], trans_w=s["trans_w"], bias=_ptr(s["bias"]), residual=_ptr(s["residual"]),
                                   pre=_ptr(s["z"]), ldx=s["x"].stride(0), ldw=s["w"].stride(0), ldy=s["y"].stride(0),
                                   ld_residual=s["residual"].stride(0) if s["residual"] is not None else 0,
                                   ld_pre=s["z"].stride(0) if s["z"] is not None else 0)
        eb.linear_device(_ptr(s["x"]), _ptr(s["w"]), _ptr(s["y"]), s["rows"], s["d_in"], s["d_out"], opts)
        return {"y": s["y"], "pre": s["z"]}
    if op == "linear_grad":
        opts = eb.make_linear_opts(dtype, activation=ACT[s["act"]], trans_w=s["trans_w"], pre=_ptr(s["z"]), ldx=s["x"].stride(0),
                                   ldw=s["w"].stride(0), ldy=s["grad_out"].stride(0), ld_pre=s["z"].stride(0) if s["z"] is not None else 0)
        eb.linear_gradients_device(_ptr(s["grad_out"]), _ptr(s["x"]), _ptr(s["w"]), _ptr(s["grad_x"]), _ptr(s["grad_w"]), _ptr(s["grad_bias"]),
                                   s["rows"], s["d_in"], s["d_out"], opts)
        return {"grad_x": s["grad_x"], "grad_w": s["grad_w"], "grad_bias": s["grad_bias"]}
    x = s["logits"]
    if op == "logprobs":
        top = s["top"]
        eb.token_logprobs_device(x.data_ptr(), _ptr(s["tokens"]), _ptr(s["logprob"]), _ptr(s["entropy"]), _ptr(s["lse"]),
                                 _ptr(s["top_logprob"]) if top else 0, _ptr(s["top_index"]) if top else 0, s["rows"], s["vocab"], top, dtype,
                                 ld=x.stride(0))
        out = {"logprob": s["logprob"], "entropy": s["entropy"], "lse": s["lse"]}
        if top:
            out["top_logprob"], out["top_index"] = s["top_logprob"], s["top_index"]
        return out
    eb.token_logprobs_gradient_device(x.data_ptr(), _ptr(s["tokens"]), _ptr(s["lse"]), _ptr(s["entropy"]), _ptr(s["grad_logprob"]),
                                      _ptr(s["grad_entropy"]), _ptr(s["grad_logits"]), s["rows"], s["vocab"], dtype, ld=x.stride(0),
                                      ld_grad=s["grad_logits"].stride(0))
    return {"grad_logits": s["grad_logits"]}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    b = BYTES[case["dtype"]]
    wide = 8 if case["dtype"] == "f64" else 4
    op, rows = case["op"], case["rows"]
    if op == "norm":
        n = case["features"]
        return {"bytes": 2 * rows * n * b + 2 * n * b + 2 * rows * wide, "flops": 8 * rows * n}
    if op == "norm_grad":
        n = case["features"]
        return {"bytes": 3 * rows * n * b + n * b + 2 * n * wide + 2 * rows * wide, "flops": 14 * rows * n}
    if op == "linear":
        k, n = case["d_in"], case["d_out"]
        outs = 1 + int(case["pre"]) + int(case["residual"])
        return {"bytes": b * (rows * k + k * n + outs * rows * n + int(case["bias"]) * n), "flops": 2 * rows * k * n}
    if op == "linear_grad":
        k, n = case["d_in"], case["d_out"]
        ins = 1 + int(case["act"] != "none")
        return {"bytes": b * (ins * rows * n + 2 * rows * k + 2 * k * n) + int(case["bias"]) * n * wide, "flops": 4 * rows * k * n}
    v = case["vocab"]
    if op == "logprobs":
        return {"bytes": rows * (v * b + 8 + 3 * wide + case["top"] * (8 + wide)), "flops": 5 * rows * v}
    return {"bytes": rows * (2 * v * b + 8 + 4 * wide), "flops": 7 * rows * v}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op == "norm":
        x = s["x"].to(f64)
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        inv = (var + EPS).rsqrt()
        return {"y": torch.addcmul(s["beta"].to(f64), (x - mean[:, None]).mul_(inv[:, None]), s["gamma"].to(f64)), "mean": mean, "inv_std": inv}
    if op == "norm_grad":
        # y = gamma xhat + beta with xhat = (x - mean) inv_std: the chain rule through mean and inv_std
        g, x, n = s["grad_out"].to(f64), s["x"].to(f64), case["features"]
        inv, mean = s["inv_std"].to(f64)[:, None], s["mean"].to(f64)[:, None]
        xhat = (x - mean).mul_(inv)
        grad_gamma, grad_beta = torch.einsum("rf,rf->f", g, xhat), g.sum(0)
        up = g.mul_(s["gamma"].to(f64))
        along = torch.einsum("rf,rf->r", up, xhat)[:, None]
        level = up.sum(1, keepdim=True)
        return {"grad_in": inv / n * (n * up - level - xhat * along), "grad_gamma": grad_gamma, "grad_beta": grad_beta}
    if op == "linear":
        w = s["w"].to(f64)
        z = torch.matmul(s["x"].to(f64), w.T if case["trans_w"] else w)
        if case["bias"]:
            z += s["bias"].to(f64)
        y = z.clamp(min=0) if case["act"] == "relu" else torch.nn.functional.gelu(z, approximate="tanh") if case["act"] == "gelu" else z
        if case["residual"]:
            y = y + s["residual"].to(f64)
        return {"y": y, "pre": z if case["pre"] else None}
    if op == "linear_grad":
        dz = s["grad_out"].to(f64)
        if case["act"] == "relu":
            dz = dz * (s["z"] > 0)
        elif case["act"] == "gelu":
            z = s["z"].to(f64)
            # with sigma the logistic function of 2 u(z): gelu = z sigma, slope = sigma + z sigma (1 - sigma) 2 u'(z)
            sigma = torch.sigmoid(2.0 * GELU_A * (z + GELU_B * z ** 3))
            dz = dz * (sigma + z * sigma * (1.0 - sigma) * 2.0 * GELU_A * (1.0 + 3.0 * GELU_B * z ** 2))
        w, x = s["w"].to(f64), s["x"].to(f64)
        grad_x = torch.matmul(dz, w if case["trans_w"] else w.T)
        grad_w = torch.matmul(dz.T, x) if case["trans_w"] else torch.matmul(x.T, dz)
        return {"grad_x": grad_x, "grad_w": grad_w, "grad_bias": dz.sum(0) if case["bias"] else None}
    rows, part = case["rows"], max(1, (1 << 27) // case["vocab"])
    done = []
    for r in range(0, rows, part):  # a part of the rows at a time: 64-bit copies of all logits would be large
        at = slice(r, min(rows, r + part))
        x, tokens = s["logits"][at].to(f64), s["tokens"][at]
        if op == "logprobs":
            lp = torch.log_softmax(x, dim=1)
            lse = torch.logsumexp(x, dim=1)
            ent = -torch.nansum(torch.special.xlogy(lp.exp(), lp.exp()), dim=1)
            logprob = torch.where(tokens >= 0, lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0.0)
            done.append((logprob, ent, lse) + ((lp.topk(case["top"], dim=1).values,) if case["top"] else ()))
        else:
            p = torch.exp(x - s["lse"][at].to(f64)[:, None])
            g = s["grad_logprob"][at].to(f64) * (tokens >= 0)
            hot = torch.zeros_like(p)
            hot.scatter_(1, tokens.clamp(min=0)[:, None], 1.0)
            inner = torch.special.xlogy(p, p) + p * s["entropy"][at].to(f64)[:, None]
            done.append((((hot - p).mul_(g[:, None])).sub_(inner.mul_(s["grad_entropy"][at].to(f64)[:, None])),))
    got = [torch.cat(parts) for parts in zip(*done)]
    if op == "logprobs_grad":
        return {"grad_logits": got[0]}
    out = {"logprob": got[0], "entropy": got[1], "lse": got[2]}
    if case["top"]:
        out["top_logprob"], out["top_index"] = got[3], None
    return out
