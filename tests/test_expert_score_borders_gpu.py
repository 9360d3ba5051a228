"""Scores that lie next to a border of fp32: the choice with a bias goes by the score in 64 bits, rounded once."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import expert_ops as ops

pytestmark = pytest.mark.gpu

# Logits (x, y) for which the score 1 / (1 + exp(x) + exp(y)) of a logit 0 beside them lies 2^-50 to 2^-47 of itself
# below a border, and the value that it rounds to.  x and y are near -ln(2) / 2, where a series of exp is least exact.
NEAR = [(-0.343849003, -0.337370008, 0.41276589), (-0.346428603, -0.329705596, 0.412142575),
        (-0.346016318, -0.341761708, 0.413561761), (-0.345827997, -0.338207096, 0.41310674),
        (-0.345328897, -0.33972612, 0.413231194), (-0.344906807, -0.34150061, 0.413395762),
        (-0.344667405, -0.328434408, 0.411775768), (-0.343479514, -0.338897318, 0.412906855),
        (-0.336135119, -0.329289109, 0.41085282), (-0.335252404, -0.327267498, 0.410500854),
        (-0.334133118, -0.3328318, 0.411040664)]


def exp(x):
    """exp of a fraction, to 2^-100."""
    s = t = Fraction(1)
    for n in range(1, 40):
        t = t * x / n
        s += t
    return s


@pytest.mark.parametrize("E", [4, 65, 200, 500, 1024])
@pytest.mark.parametrize("T", [1, 2000])
def test_scores_next_to_a_border(cuda, E, T):
    """Expert 0 has the value that the score rounds to as its bias (and the score 0): a tie, which it wins; with
    the value one step below it loses."""
    for x, y, value in NEAR:
        x, y, value = (np.float32(v) for v in (x, y, value))
        above = np.nextafter(value, np.float32(1))
        score = 1 / (1 + exp(Fraction(float(x))) + exp(Fraction(float(y))))
        border = (Fraction(float(value)) + Fraction(float(above))) / 2
        assert 0 < (border - score) / score < Fraction(1, 1 << 46)
        row = torch.full((E,), -torch.inf)
        row[1], row[2], row[E - 1] = 0.0, float(x), float(y)
        logits = row.expand(T, E).contiguous().to(cuda)
        bias = torch.full((E,), -1.0, device=cuda)
        bias[1] = 0.0
        for first, want in ((value, 0), (np.nextafter(value, np.float32(0)), 1)):
            bias[0] = float(first)
            experts, _ = ops.route_experts(logits, 1, bias=bias)
            assert (experts == want).all(), (x, y)
