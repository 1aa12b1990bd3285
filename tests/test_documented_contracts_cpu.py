"""What the public header says of rows without unmasked entries, against the definition in f64."""
import os

import numpy as np

from oracle import operators_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def header():
    with open(os.path.join(ROOT, "include", "eshkol_b200_ext.h")) as f:
        return " ".join(line.strip(" */") for line in f.read().splitlines())


def test_the_gradient_of_a_row_without_unmasked_entries():
    x = np.full((2, 5), -np.inf)
    tokens = np.array([3, -1])
    _, ent, lse = ref.token_logprobs(x, tokens, 0)[:3]
    got = ref.token_logprobs_gradient(x, tokens, lse, ent, np.array([2.0, 4.0]), np.array([1.0, 1.0]))
    assert np.array_equal(got, [[0, 0, 0, 2.0, 0], [0, 0, 0, 0, 0]])
    text = header()
    assert "a row without unmasked entries gets zeros" not in text
    assert "In a row without unmasked entries every p is 0: it gets grad_logprob at its token and zeros elsewhere." in text
