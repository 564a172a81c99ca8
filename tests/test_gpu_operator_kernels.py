'''The kernels of group norms, log probabilities and recurrences one by one: sizes that are planned for each of them, against the definitions
in 64 bits. Bounds are those of the operators' own tests.'''
import numpy as np
import pytest

from tests.test_gpu_operators import both, close, norm_bounds, norm_program
from tests.test_operators import normal

pytestmark = pytest.mark.gpu
f32 = np.float32


def check_norm(shape, groups, activation):
    print(f'group norm {shape} in {groups}, {activation}', flush=True)
    c = shape[-1]
    x, scale, shift, g = (normal(c, *shape) + normal(2, c)).astype(f32), (0.5 + np.random.default_rng(c).random(c)).astype(f32), normal(3, c, scale=0.3), normal(4, *shape)
    got, expected, closed = both(norm_program(groups, activation), x, scale, shift, g)
    for name, a, b, bound in zip(('y', 'dx', 'dscale', 'dshift'), got, expected, norm_bounds(x, scale, shift, g, groups, 1e-5, activation)):
        close(a, b, bound, name)
    return closed


@pytest.mark.parametrize('shape,groups', [((1, 3), 1), ((1, 5), 1), ((5, 255), 1), ((3000, 255), 1), ((7, 255), 3), ((1, 255), 5)])
@pytest.mark.parametrize('activation', [None, 'silu'])
def test_rows_whose_values_end_at_an_odd_word(shape, groups, activation):
    check_norm(shape, groups, activation)
