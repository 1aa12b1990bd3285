"""f32 products by bf16 parts, in numpy: what three parts hold, what fewer would lose, and that the bound of
the GPU tests on the error's norm tells the two apart."""
import numpy as np
import pytest

from eshkol_b200 import inputs
from oracle import operators_ref as ref

# the GPU tests' bound (tests/test_gpu_linear_f32.py): the hand-overs' truncations are expected to be 3.8e-7
NORM = 6e-7


@pytest.mark.parametrize("exponent", [-103, -60, 0, 60, 126])
def test_three_parts_are_the_value(exponent):
    v = ((1.0 + inputs.uniform(181, (4000,)) ** 2).clip(1.0, 1.99) * 2.0 ** exponent).astype(np.float32)
    parts = ref.bf16_parts(v)
    assert np.array_equal(sum(p.astype(np.float64) for p in parts), v.astype(np.float64))
    smallest = min(np.abs(p[p != 0]).min() for p in parts)
    assert smallest >= 2.0 ** -126  # no part below bf16's normal numbers


def test_the_products_left_out_are_at_most_2_to_the_minus_24():
    v = (1.0 + np.arange(1 << 14, dtype=np.float64) * 2.0 ** -23 * 509).astype(np.float32)
    parts = [p.astype(np.float64) for p in ref.bf16_parts(v)]
    w = v[::-1].copy()
    other = [p.astype(np.float64) for p in ref.bf16_parts(w)]
    for b, o in ((v, parts), (w, other)):
        kept = sum(parts[i] * o[j] for i in range(3) for j in range(3 - i))
        exact = v.astype(np.float64) * b.astype(np.float64)
        assert (np.abs(kept - exact) <= 2.0 ** -24 * 1.01 * exact).all()


@pytest.mark.parametrize("rows,k,n", [(64, 8192, 192), (300, 2048, 512), (777, 2001, 403)])
def test_a_missing_part_would_pass_the_bound_on_the_norm(rows, k, n):
    x, w = inputs.normal(182, (rows, k)).astype(np.float32), (inputs.normal(183, (k, n)) / np.sqrt(k)).astype(np.float32)
    want = x.astype(np.float64) @ w.astype(np.float64)
    off = [np.linalg.norm(ref.product_of_parts(x, w, c) - want) / np.linalg.norm(want) for c in (1, 2, 3)]
    assert off[2] < 0.05 * NORM  # three parts: nothing beside the sums' own rounding
    assert off[1] > 3 * NORM and off[0] > 1000 * NORM
