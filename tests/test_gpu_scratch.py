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


SCRATCH_PROGRAM = """
import sys
import torch
import eshkol_b200 as eb
lib = eb.load_library()
assert lib.eshkol_gpu_init() == 1
rows, k, n = 2000, 3000, 5000
kinds = {"f32": (torch.float32, eb.DTYPE_F32), "f16": (torch.float16, eb.DTYPE_F16)}
t, tag = kinds[sys.argv[1]]
x, w, g, z = (torch.zeros(a, b + 1, dtype=t, device="cuda")[:, :b] for a, b in ((rows, k), (k, n), (rows, n), (rows, n)))
gb = torch.empty(n, device="cuda")
torch.cuda.synchronize()
P = lambda v: v.data_ptr() if v is not None else 0
opts = eb.make_linear_opts(tag, activation=2, pre=P(z), ldx=k + 1, ldw=n + 1, ldy=n + 1, ld_pre=n + 1)
for wanted in ("b", "x", "w"):
    ox = torch.zeros(rows, k + 1, dtype=t, device="cuda")
    ow = torch.zeros(k, n + 1, dtype=t, device="cuda")
    torch.cuda.synchronize()
    eb.linear_gradients_device(P(g), P(x) if wanted == "w" else 0, P(w) if wanted == "x" else 0, P(ox) if wanted == "x" else 0,
                               P(ow) if wanted == "w" else 0, P(gb) if wanted == "b" else 0, rows, k, n, opts)
    assert eb.sync_status() == 0
    print(wanted, lib.eshkol_b200_workspace_bytes())
"""


@pytest.mark.parametrize("dtype,planes", [("f32", 3), ("f16", 1)])
def test_only_operands_of_a_product_take_scratch(gpu_lib, dtype, planes):
    """In a process of its own, whose scratch has not grown yet: the bias' gradient alone needs its partial
    sums, the gradient of x no copy of x, that of w no copy of w (partial sums of a split reduction aside)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", SCRATCH_PROGRAM, dtype], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    held = {line.split()[0]: int(line.split()[1]) for line in run.stdout.splitlines()}
    rows, k, n = 2000, 3000, 5000
    pad = lambda c: (c + 7) // 8 * 8  # noqa: E731
    dz, x, w = rows * pad(n) * 2 * planes, rows * pad(k) * 2 * planes, k * pad(n) * 2 * planes
    # partial sums of at most 512 groups of rows: 20 blocks across, and no more in all than the SMs hold
    assert held["b"] <= 512 * n * 4 + 4096, held
    # room for rounding every part up to 1024 bytes; at these sizes no reduction is split
    assert held["x"] <= dz + w + 8192, held
    assert held["w"] <= max(dz + x, dz + w) + 8192, held
