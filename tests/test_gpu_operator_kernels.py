'''The kernels of group norms, log probabilities and recurrences one by one: sizes that are planned for each of them, against the definitions
in 64 bits. Bounds are those of the operators' own tests.'''
import numpy as np
import pytest

from tests.test_gpu_operators import both, check_recurrence, close, norm_bounds, norm_program, recurrence_inputs
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


# ------------------------------------------------------------------ every kernel

#(samples, positions, groups, channels of a group): for every kernel a size at its edge (a wave or vector that is not full, a last set that is not full), and one of
#many blocks
NORM_SIZES = [(1, 5, 1, 129), (70, 13, 3, 43), (1, 17, 1, 129), (9, 31, 2, 193), (1, 2, 1, 2048), (37, 2, 1, 2048), (3, 3, 2, 1030), (75, 7, 4, 516), (1, 3, 4, 129),
              (130, 11, 4, 33), (1, 5, 4, 129), (140, 30, 8, 20), (1, 5, 2, 1030), (80, 49, 32, 16), (1, 2, 1, 4), (301, 3, 4, 4), (260, 5, 7, 3), (90, 60, 3, 20),
              (2100, 1, 2, 129), (8200, 1, 1, 129), (8191, 1, 3, 43), (1040, 1, 8, 129), (2051, 1, 16, 65), (520, 1, 32, 129), (8191, 1, 16, 65), (4099, 1, 4, 16), (3, 1, 7, 5), (1001, 1, 5, 51),
              (1, 1, 1, 1025), (77, 1, 1, 1027), (1, 1, 1, 2050), (33, 1, 2, 2051), (1100, 1, 1, 2050), (1, 1, 1, 2048), (1500, 1, 1, 2048), (5, 1, 3, 1028), (7, 1, 1, 4100), (1300, 1, 1, 2052),
              (40, 1, 1, 8200), (1025, 1, 2, 4096), (3, 1, 1, 260), (60, 1, 3, 901), (5, 1, 2, 257), (33, 2, 2, 1), (6, 900, 2, 5), (2, 5000, 3, 4), (3, 700, 1, 1300)]


@pytest.mark.parametrize('activation', ['relu', 'silu'])
@pytest.mark.parametrize('n,s,groups,cg', NORM_SIZES)
def test_every_group_norm_kernel(n, s, groups, cg, activation):
    check_norm((n, s, groups * cg) if s > 1 else (n, groups * cg), groups, activation)


#(batch, time, channels): times up to a tile's and beyond it, of whole vectors and of single channels
RECURRENCE_SIZES = [(3, 1, 8), (3, 1, 7), (2, 4, 260), (2, 4, 77), (2, 5, 1000), (1, 3, 1024), (3, 8, 512), (5, 6, 1020), (1, 16, 1024), (2, 60, 130), (40, 16, 260), (2, 8, 1001), (3, 33, 257),
                    (1, 200, 36), (1, 300, 129), (1, 1000, 132), (1, 3000, 132), (2, 5000, 31), (2, 513, 64), (1, 129, 64), (30, 2100, 64), (64, 300, 132), (9, 8, 2000), (3, 128, 4), (4, 200, 5), (3, 33, 5),
                    (2, 50, 33), (1, 33, 20), (3, 65, 20), (2, 257, 20), (1, 9000, 20), (3, 9001, 44)]


@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('b,t,c', RECURRENCE_SIZES)
def test_every_recurrence_kernel(b, t, c, gated):
    print(f'recurrence {b} x {t} x {c}, gated {gated}', flush=True)
    check_recurrence(recurrence_inputs(b, t, c, gated, True, b > 1, seed=b + t + c), gated, bool(t % 2))
