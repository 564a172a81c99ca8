'''Token models' operators on the GPU where their operands' ranges end. Tolerances as in test_gpu_token_model_operators.py.'''
import numpy as np
import pytest

from tests.test_gpu_operators import both
from tests.test_gpu_token_model_operators import orthogonal_bound
from tests.test_operators import normal
from vkjax_amd import minijax as mj

pytestmark = pytest.mark.gpu
nn = mj.nn


@pytest.mark.parametrize('steps,coefficients', [(32, (0.25, 0.0, 0.0)), (2, (0.0, 0.5, 0.0)), (2, (1e-12, 0.0, 0.0)), (1, (0.0, 0.0, 1e-20)), (5, (0.01, -0.01, 0.005))], ids=str)
@pytest.mark.parametrize('shape', [(100, 100), (70, 300), (300, 66), (40, 50)], ids=str)
def test_orthogonalize_by_polynomials_that_leave_next_to_nothing(shape, steps, coefficients):
    '''Singular values down to 1e-24: the squares of some are below what fp32 has.'''
    print(f'orthogonalize {shape}, {steps} steps, {coefficients}', flush=True)
    x = normal(5, *shape)
    (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x, steps, coefficients), x)
    expected = expected.astype(np.float64)
    off, bound = np.linalg.norm(got - expected), orthogonal_bound(x, steps, coefficients)
    assert off <= bound < 0.02 * np.linalg.norm(expected), (off, bound, np.linalg.norm(expected))
