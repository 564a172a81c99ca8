'''Token models' operators on the GPU where their operands' ranges end. Tolerances as in test_gpu_token_model_operators.py.'''
import numpy as np
import pytest

from tests.test_gpu_operators import both, close
from tests.test_gpu_token_model_operators import loss_bounds, loss_inputs, orthogonal_bound
from tests.test_operators import normal
from tests.test_token_model_operators import loss_program
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


# ------------------------------------------------------------------ log probabilities from weights

def check_masked(rows, hidden, vocabulary, transposed, mask, feature, masked, program=loss_program):
    '''Tokens that are masked by a weight of a feature that is 1 in every row: their probability is 0, and everything else is what it is without them. (Where the mask is infinite, so is what the
    feature's gradient would be: 0 times it.)'''
    print(f'masked: {rows} x {hidden} x {vocabulary}, transposed {transposed}, {mask} at feature {feature}', flush=True)
    x, w, tokens, g, gs = loss_inputs(rows, hidden, vocabulary, False)
    masked = np.asarray(masked) % vocabulary
    others = np.setdiff1d(np.arange(vocabulary), masked)
    inside = (tokens >= 0) & (tokens < vocabulary)
    tokens = np.where(inside, others[tokens % len(others)], tokens).astype(np.int32)
    tokens[0] = others[0]
    inside[0] = True
    x[:, feature] = 1
    w[feature, masked] = mask
    place = np.where(inside, np.searchsorted(others, tokens), -1)
    bounds = loss_bounds(x, w[:, others], place, g, gs, False)
    got, expected, _ = both(program(transposed), np.where(inside[:, None], x, np.nan).astype(np.float32), np.ascontiguousarray(w.T) if transposed else w, tokens, g, gs)
    for name, a, b, bound in zip(('log_probs', 'log_sums'), got, expected, bounds):
        assert np.isfinite(b).all()
        close(a, b, bound, name)
    dx, dw = got[2], got[3].T if transposed else got[3]
    expected_dx, expected_dw = expected[2], expected[3].T if transposed else expected[3]
    rest = np.arange(hidden) != feature if np.isinf(mask) else np.ones(hidden, bool)
    assert not dx[~inside].any()
    close(dx[inside][:, rest], expected_dx[inside][:, rest], bounds[2][inside][:, rest], 'dx')
    if np.isinf(mask):
        assert np.isnan(dx[inside, feature]).all()
    close(dw[:, others], expected_dw[:, others], bounds[3], 'dweights')
    assert not dw[:, masked].any()


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('hidden', [4, 41, 66, 131, 1030, 2101])
@pytest.mark.parametrize('rows', [1, 9, 40, 64])
def test_tokens_masked_by_infinite_weights_of_the_last_features(rows, hidden, transposed):
    '''Contractions that end inside a step of theirs, whose last vectors are read from further in front.'''
    for feature in (-1, -2, -4):
        check_masked(rows, hidden, 301, transposed, -np.inf, hidden + feature, [300, 299, 150, 0])
