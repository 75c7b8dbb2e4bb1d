"""Inputs at the ends of their ranges, and what torch expects of an operator, for the policy operators.

Tolerances where nothing else is said are those of test_operators_gpu.py."""
import pytest
import torch

import zeno_b200
import operators_plain as plain
from test_operators_gpu import DEV, TOL, check, gradients, inputs, matrix

pytestmark = pytest.mark.gpu


# bfloat16 updates.  32-bit work is 2e-5 off the 64-bit result at most (1.6e-4 where most directions are empty, as
# test_operators_gpu.py derives); an error e of a value takes its rounding to the neighbour in e / ulp of the cases, so
# that the squares of the differences add to e ulp, with an ulp of 2^-7 of the value at most: sqrt(2e-5 * 2^-7) = 4e-4 and
# sqrt(1.6e-4 * 2^-7) = 1.2e-3 against the 64-bit result rounded to bfloat16.
@pytest.mark.parametrize("shape", [(64, 29), (128, 512), (129, 300), (200, 513), (512, 1024), (3, 260, 140), (1100, 700)])
def test_orthogonalize_bfloat16_as_32_bits_rounded_once(shape):
    m = matrix(shape, torch.bfloat16, seed=1)
    assert plain.off(zeno_b200.orthogonalize(m), plain.orthogonalize(m).bfloat16()) <= 4e-4


@pytest.mark.parametrize("shape", [(60, 90), (200, 300), (512, 1024), (700, 150)])
def test_orthogonalize_bfloat16_of_low_rank(shape):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    left, right = (torch.randint(-1, 2, s, generator=gen, device=DEV).float() for s in ((shape[0], 4), (4, shape[1])))
    m = (left @ right).bfloat16()  # whole numbers up to 4: of rank 4 to the last bit
    assert plain.off(zeno_b200.orthogonalize(m), plain.orthogonalize(m).bfloat16()) <= 1.2e-3
