'''The kernels of group norms, log probabilities and recurrences one by one: sizes that are planned for each of them, against the definitions
in 64 bits. Bounds are those of the operators' own tests.'''
import ctypes

import numpy as np
import pytest

import vkjax_amd
from tests.test_gpu_operators import D, U, both, check_recurrence, close, norm_bounds, norm_program, probs_program, recurrence_inputs
from tests.test_operator_plans import norm_launches
from tests.test_operators import normal
from vkjax_amd import hip, kernels as K, minijax as mj

pytestmark = pytest.mark.gpu
jnp, lax, nn, f32 = mj.numpy, mj.lax, mj.nn, np.float32


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


# ------------------------------------------------------------------ the gradient of log probabilities at scores far from zero

@pytest.mark.parametrize('rows,v', [(6, 40), (700, 37), (9, 900), (1200, 3500), (5, 9001), (3, 60001)])
@pytest.mark.parametrize('offset', [0.0, 100.0, -3e4, 3e4, 1e6])
def test_log_probs_gradient_does_not_go_by_a_rounded_log_of_the_sum(rows, v, offset):
    print(f'gradient of log probabilities {rows} x {v} around {offset}', flush=True)
    rng = np.random.default_rng(rows + v)
    z, t = (normal(1, rows, v, scale=2.5) + f32(offset)).astype(f32), rng.integers(0, v, rows).astype(np.int32)
    t[1] = -1
    g = [np.abs(normal(11, rows)) + f32(0.5), normal(12, rows), normal(13, rows, 3)]
    got, expected, _ = both(probs_program(3), z, t, *g)
    z64 = z.astype(np.float64)
    best = z64.max(axis=1, keepdims=True)
    e = np.exp(z64 - best)
    s = e.sum(axis=1, keepdims=True)
    p, spread, log_s = e / s, best - z64, np.log(s)
    #log p = (x - (the log of the sum, rounded)) - its rest: their sum is m + log s to the last bit, log s off by the sum's error (every term by 4 u and
    #by the roundings of its exponent, then added up) and the logarithm's 2 u; the two differences are rounded. Nothing of that goes with |m|.
    mean_spread = (p * spread).sum(axis=1, keepdims=True)
    e_s = (D + 6) * U + 3 * U * mean_spread
    logp = spread + log_s
    e_lp = e_s + 2 * U * log_s + 2 * U * (logp + log_s + 1)
    mean_square = (p * spread ** 2).sum(axis=1, keepdims=True)
    e_h = e_s * (1 + 2 * mean_spread) + ((D + 8) * mean_spread + 3 * mean_square) * U + 8 * U * (log_s + mean_spread + 1)
    e_p = p * (e_lp + (3 * logp + 8) * U)
    total, gh, entropy = sum(np.abs(a.reshape(rows, -1)).sum(axis=1, keepdims=True) for a in g), np.abs(g[1])[:, None], log_s + mean_spread
    own = np.zeros_like(p)
    np.put_along_axis(own, np.maximum(t, 0)[:, None], 1.0, 1)
    for k in range(3):
        np.put_along_axis(own, got[3][:, k:k + 1].clip(0).astype(np.int64), 1.0, 1)
    e_d = e_p * (total + gh * (logp + entropy)) + p * (44 * U * total + gh * (e_lp + e_h + 4 * U * (logp + entropy))) + 8 * U * total * (own + p)
    close(got[-1], expected[-1], e_d + 1e-37, 'gradient')
    #cotangents of log probabilities alone: a row's gradient adds up to nothing, off by as much as its terms
    (d,), _, _ = both(lambda z, t, g: mj.vjp(lambda v: nn.token_log_probs(v, t)[0], z)[1](g), z, t, g[0])
    assert (np.abs(d.astype(np.float64).sum(axis=1)) <= (e_p * g[0][:, None] + 8 * U * p * g[0][:, None]).sum(axis=1) + 2 * U * g[0]).all()


@pytest.mark.parametrize('v', [30, 2000, 40000])
def test_log_probs_of_rows_that_hold_the_lowest_value_only(v):
    '''A mask of the type's lowest value that leaves nothing: such rows have a distribution, the same for every score.'''
    z = np.full((3, v), np.finfo(f32).min, f32)
    z[1, 3] = 0.0
    t, g = np.array([0, 3, v - 1], np.int32), np.ones(3, f32)
    lp, entropy, d = both(lambda z, t, g: (lambda outs, pull: outs + pull((g, g)))(*mj.vjp(lambda q: nn.token_log_probs(q, t), z)), z, t, g)[0]
    one = np.zeros(v)
    close(lp, [-np.log(v), 0, -np.log(v)], 8 * U * np.log(v))
    close(entropy, [np.log(v), 0, np.log(v)], 8 * U * np.log(v))
    for row, token in ((0, 0), (2, v - 1)):
        one[:] = 0
        one[token] = 1
        #(the entropy of equal probabilities has no gradient: what is left of it is log p + H, off by 16 u log v)
        close(d[row], one - 1 / v, (24 * U * np.log(v) + 16 * U) / v + 2 * U * one)
    assert not d[1].any()


# ------------------------------------------------------------------ the relu of the forward pass and that of the gradient

#(samples, positions, groups, channels of a group): both directions in registers, in chunks, forward in registers and the gradient in chunks, rows, wide rows, forward
#wide and the gradient in chunks
@pytest.mark.parametrize('n,s,groups,cg,kinds', [(2, 49, 64, 16, ('held', 'held')), (3, 17, 5, 129, ('held', 'held')), (1, 4000, 32, 16, ('chunked', 'chunked')), (1, 4001, 7, 33, ('chunked', 'chunked')),
                                                 (80, 49, 32, 16, ('held', 'held')), (70, 1200, 4, 8, ('held', 'chunked')), (24, 1, 16, 65, ('rows', 'rows')), (24, 1, 2, 2048, ('wide', 'wide')),
                                                 (24, 1, 1, 20000, ('wide', 'chunked'))])
def test_the_gradient_goes_through_where_the_result_is_positive(n, s, groups, cg, kinds):
    '''Every channel's shift puts one of its values next to zero; the cotangents are 1, 2, 4 .., so that the shift's gradient tells which values went through.'''
    c = groups * cg
    assert tuple(K.norm_plan(n, s, c, groups, gradient).kind for gradient in (False, True)) == kinds
    shape = (n, s, c) if s > 1 else (n, c)
    x, scale = (normal(c, *shape) + normal(2, c)).astype(f32), (0.5 + np.random.default_rng(c).random(c)).astype(f32)
    _, mean, rstd = vkjax_amd.wrap(lambda *a: lax.group_norm(*a, groups), frontend='minijax')(x, scale, np.zeros(c, f32))
    rows, places = x.reshape(n * s, c), 20
    which = np.arange(c) % places
    sample, group = which // s, np.arange(c) // cg
    hat = (rows[which, np.arange(c)] - mean[sample, group]) * rstd[sample, group]
    shift = -(hat * scale)
    g = np.zeros((n * s, c), f32)
    g[:places] = 2.0 ** np.arange(places)[:, None]
    y, _, _, dshift = vkjax_amd.wrap(norm_program(groups, 'relu'), frontend='minijax')(x, scale, shift, g.reshape(shape))
    passed = (y.reshape(n * s, c)[:places] > 0) * g[:places].astype(np.float64)
    assert np.array_equal(dshift, passed.sum(axis=0)), int((dshift != passed.sum(axis=0)).sum())


# ------------------------------------------------------------------ recurrences whose products of factors leave the range of fp32

@pytest.mark.parametrize('t,c', [(40, 8), (700, 12), (700, 7), (3000, 20)])
@pytest.mark.parametrize('gated,reverse', [(False, False), (True, True)])
def test_recurrences_behind_many_small_factors(gated, reverse, t, c):
    '''A state of 1e38 behind which products of factors fall below 2^-149: an error of 2^-140 of it; an infinite one leaves no finite value in its channel, and
    the others as they are.'''
    print(f'recurrence 2 x {t} x {c}, gated {gated}, small factors', flush=True)
    x, state = np.abs(normal(1, 2, t, c)), np.zeros((2, c), f32)
    factor = np.full((2, t, c), -1.5 if gated else 0.25, f32)
    state[0, 1::2] = 1e38
    got, expected, _ = both(lambda *a: (nn.gated_recurrence if gated else lax.linear_recurrence)(*a, reverse=reverse), factor, x, state)
    #24 u a step of what is kept, of a geometric series (below twice its largest term) of values of at most 6, and of the state
    a = 1 / (1 + np.exp(1.5)) if gated else 0.25
    left = np.abs(state[:, None].astype(np.float64)) * a ** np.arange(1, t + 1)[None, :, None]
    left = left[:, ::-1] if reverse else left
    steps = np.arange(1, t + 1)[None, :, None]
    steps = steps[:, ::-1] if reverse else steps
    for k, bound in ((0, 24 * U * (12 + steps * left) + 2.0 ** -140 * np.abs(state[:, None])), (1, 24 * U * (12 + t * left[:, 0 if reverse else -1]) + 2.0 ** -140 * np.abs(state))):
        close(got[k], expected[k], bound + 1e-37, ('h', 'last')[k])
    state[0, 0] = np.inf
    broken, _, _ = both(lambda *a: (nn.gated_recurrence if gated else lax.linear_recurrence)(*a, reverse=reverse), factor, x, state)
    assert not np.isfinite(broken[0][0, :, 0]).any() and not np.isfinite(broken[1][0, 0])
    broken[0][0, :, 0], broken[1][0, 0] = got[0][0, :, 0], got[1][0, 0]
    assert np.array_equal(broken[0], got[0]) and np.array_equal(broken[1], got[1])


# ------------------------------------------------------------------ beside other users of the runtime

def test_looking_for_a_kernel_leaves_no_error_behind():
    '''The kernel is in the last of the modules that are searched: the searches that fail are nobody's error.'''
    runtime = ctypes.CDLL('libamdhip64.so.7')
    runtime.hipGetLastError()
    device = hip.Device(hip.Device.get().index)
    f = vkjax_amd.wrap(lambda a, x: lax.linear_recurrence(a, x)[0], frontend='minijax', device=device)
    h = f(np.full((1, 3, 4), 0.5, f32), np.ones((1, 3, 4), f32))
    assert runtime.hipPeekAtLastError() == 0 and np.array_equal(h[0, :, 0], [1, 1.5, 1.75])


# ------------------------------------------------------------------ more rows than 24 bits count

@pytest.mark.parametrize('v,top', [(20, 0), (124, 5)])
def test_log_probs_of_more_rows_than_a_block_each_can_be_launched_for(v, top):
    rows = 2**24 + 5
    print(f'log probabilities {rows} x {v}, top {top}', flush=True)
    row, t = normal(v, v), (np.arange(rows) % v).astype(np.int32)
    t[3], t[rows - 2] = -1, v
    got = vkjax_amd.wrap(lambda row, t: nn.token_log_probs(jnp.broadcast_to(jnp.reshape(row, (1, v)), (rows, v)), t, top)[:3], frontend='minijax')(row, t)
    logp = row.astype(np.float64)
    logp = logp - (logp.max() + np.log(np.exp(logp - logp.max()).sum()))
    #sums of at most 64 additions in a row, twice over, and roundings of values of at most 20
    bound = 160 * U + 6 * U * 20
    given = (t >= 0) & (t < v)
    expected = np.where(given, logp[np.where(given, t, 0)], 0.0)
    close(got[0], expected, bound)
    close(got[1], np.where(given, -(np.exp(logp) * logp).sum(), 0.0), 20 * bound)
    if top:
        close(got[2][-9:], np.where(given[-9:, None], np.sort(logp)[::-1][:top], 0.0), bound)


# ------------------------------------------------------------------ single steps of more than two gigabytes

def test_single_steps_of_more_than_two_gigabytes():
    b, c = 2**19 + 3, 1020
    gate, x, state = normal(1, c), normal(2, b), normal(3, b)

    def f(gate, x, state):
        spread = lambda v: jnp.broadcast_to(jnp.reshape(v, (b, 1, 1)), (b, 1, c))
        start = jnp.broadcast_to(jnp.reshape(state, (b, 1)), (b, c))
        h, last = nn.gated_recurrence(jnp.broadcast_to(jnp.reshape(gate, (1, 1, c)), (b, 1, c)), spread(x), start)
        return h[b - 7:, 0], last[b // 2 - 3:b // 2 + 3], h[:5, 0]
    a = 1 / (1 + np.exp(-gate.astype(np.float64)))
    exact = lambda part: a * state[part, None].astype(np.float64) + (1 - a) * x[part, None].astype(np.float64)
    for got, part in zip(vkjax_amd.wrap(f, frontend='minijax')(gate, x, state), (slice(b - 7, b), slice(b // 2 - 3, b // 2 + 3), slice(0, 5))):
        close(got, exact(part), 24 * U * (np.abs(state[part, None]) + np.abs(x[part, None])))


# ------------------------------------------------------------------ many samples of few positions with wide groups: one row of channel sums for several of them

@pytest.mark.parametrize('n,s,groups,cg', [(700, 1, 1, 16388), (643, 2, 1, 8195), (1300, 3, 1, 4100), (601, 1, 1, 8197), (259, 15, 1, 16500), (900, 1, 2, 16500)])
def test_chunked_samples_that_share_a_row_of_sums(n, s, groups, cg):
    c = groups * cg
    backward = norm_launches(n, s, groups, cg)[1]
    assert K.norm_plan(n, s, c, groups, True).kind == 'chunked' and backward[0].grid[0] < n * K.norm_plan(n, s, c, groups, True).spans
    check_norm((n, s, c) if s > 1 else (n, c), groups, 'silu')
