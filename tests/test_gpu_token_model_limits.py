'''Token models' operators on the GPU where their operands' ranges end. Tolerances as in test_gpu_token_model_operators.py.'''
import numpy as np
import pytest

import tests.test_gpu_token_model_operators as operators
from tests.test_gpu_operators import U, both, close
from tests.test_gpu_token_model_operators import loss_bounds, loss_inputs, orthogonal_bound
from tests.test_operators import normal
from tests.test_token_model_operators import loss_program, scan_inputs, scan_program
from vkjax_amd import kernels as K, minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

pytestmark = pytest.mark.gpu
lax, nn = mj.lax, mj.nn
f32 = np.float32


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


@pytest.fixture
def fp32_products(monkeypatch):
    '''Bounds of products of more than 64 rows where their operands are too far apart for the fp16 matrix cores: one sum after the other, rounded for every term, at most twice where it is put
    together from slices.'''
    monkeypatch.setattr(operators, 'product_error', lambda a, b, terms: (terms + 70) * U * (a @ b))


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('mask', [-np.inf, -1e30, -3.4e38, -1e9])
@pytest.mark.parametrize('rows,hidden,vocabulary', [(65, 41, 301), (70, 3, 200), (150, 131, 1300), (300, 64, 2049), (20, 2, 30)])
def test_tokens_masked_by_weights_of_any_size(rows, hidden, vocabulary, mask, transposed, fp32_products):
    for feature in (0, hidden - 1):
        check_masked(rows, hidden, vocabulary, transposed, mask, feature, [0, 7, vocabulary - 1, vocabulary - 2])


@pytest.mark.parametrize('slices', [1, 3])
@pytest.mark.parametrize('kernel,side', [(k[0], k[1]) for k in K.HALF_KERNELS])
def test_tokens_masked_in_every_kernel_of_a_product(kernel, side, slices, monkeypatch, fp32_products):
    monkeypatch.setattr(K, 'half_plan', lambda tiles_of, pairs: K.HalfPlan(kernel, side, 3 if slices > 1 else tiles_of(side), min(slices, pairs)))
    for transposed in (False, True):
        check_masked(700, 300, 1500, transposed, -1e30, 17, [0, 129, 1499])


@pytest.mark.parametrize('transposed', [False, True])
def test_tokens_masked_in_pieces_of_the_vocabulary(transposed, monkeypatch, fp32_products):
    monkeypatch.setattr(K, 'LINEAR_PIECE', 1)
    for rows, hidden, vocabulary in ((140, 70, 600), (520, 33, 300)):
        check_masked(rows, hidden, vocabulary, transposed, -np.inf, 5, [0, 200, vocabulary - 1])


def without_parts(transposed):
    def f(x, w, tokens, g, gs):
        outs = lax.linear_log_probs(x, w, tokens, transposed)
        return outs[:2] + lax.linear_log_probs_grad(x, w, tokens, outs[2], outs[3], g, gs, transposed)
    return f


@pytest.mark.parametrize('transposed', [False, True])
def test_tokens_masked_where_nothing_was_kept(transposed, fp32_products):
    check_masked(150, 70, 600, transposed, -1e30, 5, [0, 200, 599], without_parts)


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('size', [1e12, 1e20, 1e30])
@pytest.mark.parametrize('rows', [30, 90, 400])
def test_rows_beside_one_that_is_much_larger(rows, size, transposed, fp32_products):
    '''The other rows are as exact as without it. Its own probabilities are 1 and 0 (scores lie apart by far more than they are off by), so that it adds to two tokens' weights alone.'''
    x, w, tokens, g, gs = loss_inputs(rows, 70, 500, transposed)
    tokens[:6] = np.arange(6)
    x[5] *= f32(size)
    got, expected, _ = both(loss_program(transposed), x, w, tokens, g, gs)
    w64 = (w.T if transposed else w).astype(np.float64)
    scores, others = x[5].astype(np.float64) @ w64, np.arange(rows) != 5
    top = scores.argmax()
    rounding = 140 * U * np.abs(x[5].astype(np.float64)) @ np.abs(w64)
    assert top != tokens[5] and np.diff(np.sort(scores))[-1] > 1e3 * rounding.max()
    bounds = loss_bounds(x, w, np.where(others, tokens, -1), g, gs, transposed)
    for name, a, b, bound in zip(('log_probs', 'log_sums', 'dx'), got, expected, bounds):
        close(a[others], b[others], bound[others], name)
    close(got[0][5], expected[0][5], rounding[5] + rounding[top])
    close(got[1][5], expected[1][5], rounding[top])
    ds = {tokens[5]: abs(float(g[5])), top: abs(float(gs[5]) - float(g[5]))}
    close(got[2][5], expected[2][5], 8 * U * sum(d * np.abs(w64[:, v]) for v, d in ds.items()))
    own = np.zeros((500, 70))
    for v, d in ds.items():
        own[v] = 8 * U * d * np.abs(x[5].astype(np.float64))
    close(got[3], expected[3], bounds[3] + (own if transposed else own.T), 'dweights')


def test_cotangents_of_rows_that_are_much_larger(fp32_products):
    #a row's own factor: the gradient of another row is what it is without it
    x, w, tokens, g, gs = loss_inputs(90, 70, 500, False)
    tokens[:6] = np.arange(6)
    x[4] *= f32(1e15)
    g[5], gs[5] = f32(1e15), f32(-1e12)
    got, expected, _ = both(loss_program(False), x, w, tokens, g, gs)
    for name, a, b, bound in zip(('log_probs', 'log_sums', 'dx', 'dweights'), got, expected, loss_bounds(x, w, tokens, g, gs, False)):
        close(a, b, bound, name)


@pytest.mark.parametrize('power', [9, 10, 11])
def test_scores_where_products_change(power, monkeypatch):
    '''Largest numbers whose products with one another and with the number of features are at 2^26: either kind of product, whose bounds are added up.'''
    one = operators.product_error
    monkeypatch.setattr(operators, 'product_error', lambda a, b, terms: one(a, b, terms) + (terms + 70) * U * (a @ b))
    x, w, tokens, g, gs = loss_inputs(100, 64, 400, False)
    tokens[tokens == 9] = 8
    x[:, 3], w[3] = 2.0 ** 10, 0.0
    w[3, 9] = -2.0 ** power
    got, expected, _ = both(loss_program(False), x, w, tokens, g, gs)
    bounds = loss_bounds(x, w, tokens, g, gs, False)
    for name, a, b, bound in zip(('log_probs', 'log_sums', 'dx', 'dweights'), got, expected, bounds):
        close(a, b, bound, name)


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('graph', [False, True])
def test_one_program_for_numbers_near_and_far(graph, transposed):
    near = loss_inputs(150, 70, 600, transposed)
    far = [v.copy() for v in near]
    far[0][3] *= f32(1e25)
    infinite = [v.copy() for v in near]
    infinite[1][(8, 4) if transposed else (4, 8)] = np.inf
    program = JaxprInterpreter(mj.make_jaxpr(loss_program(transposed))(*near), graph=graph)
    alone = [JaxprInterpreter(mj.make_jaxpr(loss_program(transposed))(*v)).run(*v) for v in (near, far, infinite)]
    assert np.isfinite(alone[0][3]).all() and not np.array_equal(alone[0][0], alone[1][0])
    for which in (0, 1, 0, 2, 2, 0, 1, 1, 0):
        values = (near, far, infinite)[which]
        if graph:
            program.upload_inputs(*values)
            program.replay(2)
            got = program.read_outputs()
        else:
            got = program.run(*values)
        for a, b in zip(got, alone[which]):
            assert np.array_equal(np.asarray(a).reshape(b.shape), b, equal_nan=True)


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('rows', [9, 40, 64, 65, 200])
def test_infinite_weights_are_those_of_fp32_arithmetic(rows, transposed):
    '''A score is infinite, and its probability 0, 1 or NaN, whatever the number of rows.'''
    x, w, tokens, g, gs = loss_inputs(rows, 41, 300, transposed)
    tokens[:] = np.arange(rows) % 7
    x[::3, 7], x[1::3, 7], x[2::3, 7] = 1.0, -1.0, 0.0
    for value in (np.inf, -np.inf):
        w[(9, 7) if transposed else (7, 9)] = value
        got, expected, _ = both(loss_program(transposed), x, w, tokens, g, gs)
        fine = np.sign(x[:, 7]) == -np.sign(value)
        assert np.array_equal(np.isfinite(expected[0]), fine)
        for name, a, b in zip(('log_probs', 'log_sums', 'dx'), got, expected):
            assert np.array_equal(np.isfinite(a), np.isfinite(b)), name
        (w if transposed else w.T)[9, 7] = 0
        bounds = loss_bounds(np.where(np.arange(41) == 7, 0, x).astype(f32), np.delete(w, 9, 0 if transposed else 1), tokens, g, gs, transposed)
        for a, b, bound in zip(got[:2], expected, bounds):
            close(a[fine], b[fine], bound[fine] + 41 * U * np.abs(b[fine]))


# ------------------------------------------------------------------ selective scans

@pytest.mark.parametrize('n', [3, 7, 16, 30, 64])
@pytest.mark.parametrize('time', [5, 300])
def test_scans_whose_last_step_is_infinite(time, n):
    '''A state that becomes infinite in the last step of a sequence is that behind its length too; a cotangent that does in the gradient's first step is what goes on from there (where time is
    not cut: products of many factors may be 0, and NaN times that).'''
    arrays, g, g_last = scan_inputs(3, time, 64, n, (), False)
    lengths = np.array([time, time // 2 + 1, 3], np.int32)
    for name in ('b', 'c'):
        spoiled = {k: v.copy() for k, v in arrays.items()}
        for i, end in enumerate(lengths):
            spoiled[name][i, end - 1, 1] = np.inf
        got, expected, _ = both(scan_program(list(arrays), lengths, False), g, g_last, *spoiled.values())
        outs = dict(zip(['y', 'last', *arrays], zip(got, expected)))
        for result in ('y', 'last') + (('x', 'b', 'c') if name == 'c' and time < 8 else ()):
            a, b = outs[result]
            assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.sign(a[np.isinf(b)]), np.sign(b[np.isinf(b)])) and np.array_equal(np.isinf(a), np.isinf(b)), (name, result)
        a, b = outs['last']
        assert not np.isnan(a).any() and (np.isinf(a[:, :, 1]).all() if name == 'b' else np.isfinite(a).all())


# ------------------------------------------------------------------ orthogonalised matrices of any size

@pytest.mark.parametrize('scale,eps', [(1e-37, 1e-38), (1e-30, 1e-36), (1e-25, 1e-30), (1e-22, 1e-45), (1e-19, 1e-7), (1e18, 1e-7), (1e22, 1e-7), (1e37, 1e-7), (8e37, 1e30)])
@pytest.mark.parametrize('shape', [(100, 100), (70, 300), (300, 70), (2, 65, 3), (2, 3, 1200), (40, 50)], ids=str)
def test_orthogonalize_by_the_norm_of_its_matrix(shape, scale, eps):
    '''Squares that fp32 does not have, either way; a norm beside which eps is nothing, or the other way round.'''
    if min(shape[-2:]) in range(4, 65) and not 1e-36 < scale < 1e35:
        scale = 1e-35 if scale < 1 else 1e34
    x = normal(7, *shape)
    x *= f32(min(scale, 3.2e38 / float(np.abs(x).max())))
    (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x, 3, (1.5, -0.5, 0.0), eps), x)
    for a, b, m in zip(got.reshape(-1, *shape[-2:]), expected.reshape(-1, *shape[-2:]), x.reshape(-1, *shape[-2:])):
        off, bound = np.linalg.norm(a.astype(np.float64) - b), orthogonal_bound(m, 3, (1.5, -0.5, 0.0), float(f32(eps)))
        assert off <= bound, (off, bound, np.linalg.norm(b.astype(np.float64)))


@pytest.mark.parametrize('steps,coefficients', [(1, (3.4445, -4.7750, 2.0315)), (5, (3.4445, -4.7750, 2.0315)), (32, (1.5, -0.5, 0.0)), (4, (0.1, 0.0, 0.0)), (10, (2.0, -1.5, 0.5)), (9, (3.4445, -4.7750, 2.0315))], ids=str)
@pytest.mark.parametrize('shape', [(100, 100), (70, 300), (300, 70), (3, 1200), (40, 50)], ids=str)
def test_orthogonalize_matrices_that_eps_leaves_small(shape, steps, coefficients):
    '''Norms far below eps: a stack of matrices, of which each has the bits that it has by itself, whatever the steps raise it to.'''
    sizes = np.array([1.0, 1e-3, 1e-5, 1e-8, 1e-12, 1e-17, 1e-25, 0.0])
    x = (normal(8, len(sizes), *shape) * sizes[:, None, None]).astype(f32)
    (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x, steps, coefficients, 1.0), x)
    assert not got[-1].any()
    for a, b, m in zip(got[:-1], expected, x):
        off, bound = np.linalg.norm(a.astype(np.float64) - b), orthogonal_bound(m, steps, coefficients, 1.0)
        assert off <= bound, (off, bound, np.linalg.norm(b.astype(np.float64)))


def test_orthogonalize_a_matrix_that_is_not_finite():
    for value in (np.inf, -np.inf, np.nan):
        for rows, columns in ((150, 90), (40, 90), (3, 70)):
            x = normal(1, 3, rows, columns)
            x[1, rows // 2, 5] = value
            got, = JaxprInterpreter(mj.make_jaxpr(lambda x: nn.orthogonalize(x))(x)).run(x)
            assert np.isnan(got[1]).all() and np.isfinite(got[0]).all() and np.isfinite(got[2]).all()
