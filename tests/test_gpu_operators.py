'''Group norm, log probabilities of tokens and linear recurrences on the GPU against their definitions in 64 bits (the oracle), at the
sizes, masks and paddings where they can go wrong.

Tolerances. u = 2^-24 is half a step of fp32. A sum in these kernels ends after at most D = 64 additions one after the other at the
sizes below (in a thread, then across threads), so it is off by at most D u times the sum of its terms' magnitudes; every other step
is off by u, and the exponential and the division by at most 4 u (the device library's bounds).'''
import numpy as np
import pytest

import vkjax_amd
from oracle.eval_jaxpr import eval_closed_jaxpr
from tests.test_operators import normal, token_model_inputs, token_model_step
from vkjax_amd import minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

pytestmark = pytest.mark.gpu
jnp, lax, nn = mj.numpy, mj.lax, mj.nn
f32, U, D = np.float32, 2.0 ** -24, 64


def both(f, *args, **kwargs):
    '''Results of the device and of the oracle.'''
    got = vkjax_amd.wrap(f, frontend='minijax', **kwargs)(*args)
    closed = mj.make_jaxpr(f)(*args)
    return mj.tree_leaves(got), eval_closed_jaxpr(closed, *mj.tree_leaves(args)), closed


def close(a, b, bound, what=''):
    '''|a - b| <= bound everywhere, and what is not finite is the same.'''
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    assert a.shape == b.shape, (what, a.shape, b.shape)
    fine = np.isfinite(b)
    assert np.array_equal(a[~fine], b[~fine], equal_nan=True), (what, a[~fine][:4], b[~fine][:4])
    bound = np.broadcast_to(np.asarray(bound, np.float64), b.shape)[fine]
    off = np.abs(a[fine] - b[fine])
    assert (off <= bound).all(), (what, float((off / np.maximum(bound, 1e-300)).max()), int((off > bound).sum()))


# ------------------------------------------------------------------ group norm

def norm_program(groups, activation, eps=1e-5):
    def f(x, scale, shift, g):
        y, pullback = mj.vjp(lambda *a: nn.group_norm(*a, groups, eps, activation), x, scale, shift)
        return (y,) + pullback(g)
    return f


def norm_bounds(x, scale, shift, g, groups, eps, activation):
    '''How far y, dx, dscale and dshift may be off.'''
    n, c = x.shape[0], x.shape[-1]
    x64 = x.astype(np.float64).reshape(n, -1, groups, c // groups)
    mean = x64.mean(axis=(1, 3), keepdims=True)
    var = ((x64 - mean) ** 2).mean(axis=(1, 3), keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    size = np.abs(x64).mean(axis=(1, 3), keepdims=True)
    hat = (x64 - mean) * rstd
    gamma, beta = np.abs(scale.astype(np.float64)).reshape(groups, -1), np.abs(shift.astype(np.float64)).reshape(groups, -1)
    #the mean is off by D u times the mean magnitude, hat by that times rstd (twice: the variance of deviations from a mean that
    #is off by e is off by e^2, far less), by D u of itself through the variance (half of its D u) and by a few roundings
    e_mean = (D + 2) * U * size * rstd
    e_hat = e_mean + (D / 2 + 8) * U * np.abs(hat) + 2 * U * (np.abs(x64) + np.abs(mean)) * rstd
    z = hat * scale.astype(np.float64).reshape(groups, -1) + shift.astype(np.float64).reshape(groups, -1)
    e_z = e_hat * gamma + 3 * U * (np.abs(hat) * gamma + beta)
    #the activations' slopes are at most 1.1, and they add a few roundings of their results (silu: an exponential and a division)
    e_y = 1.1 * e_z + 12 * U * np.abs(z) + 1e-37
    #act' changes by at most half of e_z (silu); where a relu's input is that near to zero it may come out on the other side
    d = np.abs(g.astype(np.float64).reshape(x64.shape)) * 1.1
    e_d = d * (e_z + 24 * U) if activation == 'silu' else d * ((np.abs(z) <= e_z) if activation == 'relu' else 0) + d * U
    count = x64.shape[1]
    sums = lambda v: v.sum(axis=(0, 1)).reshape(-1)
    e_shift = sums(e_d + (D + 2) * U * d)
    e_scale = sums(e_d * np.abs(hat) + d * e_hat + (D + 4) * U * d * np.abs(hat))
    over = lambda v: v.mean(axis=(1, 3), keepdims=True)
    ds, e_ds = d * gamma, e_d * gamma + 2 * U * d * gamma
    m1, e_m1 = over(ds), over(e_ds) + (D + 4) * U * over(ds)
    m2, e_m2 = over(ds * np.abs(hat)), over(e_ds * np.abs(hat) + ds * e_hat) + (D + 4) * U * over(ds * np.abs(hat))
    inner = ds + m1 + np.abs(hat) * m2
    e_dx = rstd * (e_ds + e_m1 + e_hat * m2 + np.abs(hat) * e_m2 + 6 * U * inner) + (D / 2 + 8) * U * rstd * inner
    return [v.reshape(x.shape) for v in (e_y, e_dx)] + [e_scale + 1e-37, e_shift + 1e-37]


#(shape, groups): one position and many, odd numbers of everything, one channel to a group, one group, groups of no multiple of 4,
#few samples with many positions and many samples with few, a wide last axis
NORMS = [((1, 1, 1, 1), 1), ((1, 4), 1), ((1, 7, 7, 512), 32), ((3, 5, 4, 6), 3), ((2, 9, 33), 11), ((5, 1, 40), 8), ((2, 56, 56, 64), 32),
         ((4, 17, 13, 24), 24), ((3, 31, 29, 20), 1), ((1, 100, 100, 8), 2), ((700, 48), 4), ((257, 1040), 16), ((9, 3, 2052), 4), ((2, 640, 7), 7),
         ((6, 11, 130), 2), ((1, 3, 4100), 1), ((33, 16, 16, 3), 3), ((2, 25, 25, 96), 32), ((5, 8191), 1), ((3, 2, 1024), 1024)]


@pytest.mark.parametrize('activation', [None, 'relu', 'silu'])
@pytest.mark.parametrize('shape,groups', NORMS, ids=[f'{s}-{g}' for s, g in NORMS])
def test_group_norm_and_gradient(shape, groups, activation):
    print(f'group norm {shape} in {groups}, {activation}', flush=True)
    rng = np.random.default_rng(len(shape) * 1000 + shape[-1])
    c = shape[-1]
    x = (normal(1, *shape) * (0.5 + rng.random(c)) + normal(2, c)).astype(f32)
    scale, shift, g = (0.5 + rng.random(c)).astype(f32), normal(3, c, scale=0.3), normal(4, *shape)
    got, expected, _ = both(norm_program(groups, activation), x, scale, shift, g)
    for name, a, b, bound in zip(('y', 'dx', 'dscale', 'dshift'), got, expected, norm_bounds(x, scale, shift, g, groups, 1e-5, activation)):
        close(a, b, bound, name)


def test_group_norm_of_values_far_from_zero_and_of_constants():
    #a variance that a difference of squares would lose; a group without any variance
    x = (1000.0 + 0.01 * normal(1, 2, 20, 20, 16)).astype(f32)
    x[1] = 7.0
    scale, shift, g = np.ones(16, f32), normal(2, 16), normal(3, 2, 20, 20, 16)
    got, expected, _ = both(norm_program(4, None), x, scale, shift, g)
    bounds = norm_bounds(x, scale, shift, g, 4, 1e-5, None)
    for name, a, b, bound in zip(('y', 'dx', 'dscale', 'dshift'), got, expected, bounds):
        close(a, b, bound, name)


def test_group_norm_keeps_a_broken_sample_to_itself():
    x = normal(1, 4, 6, 6, 8)
    x[1, 2, 3, 1], x[2, 0, 0, 7] = np.nan, np.inf
    f = vkjax_amd.wrap(lambda x, s, b: nn.group_norm(x, s, b, 2, activation='relu'), frontend='minijax')
    y = f(x, np.ones(8, f32), np.zeros(8, f32))
    clean = f(np.where(np.isfinite(x), x, f32(0)), np.ones(8, f32), np.zeros(8, f32))
    assert np.isnan(y[1, ..., :4]).all() and np.isnan(y[2, ..., 4:]).all()
    for sample, part in ((0, slice(0, 8)), (1, slice(4, 8)), (2, slice(0, 4)), (3, slice(0, 8))):
        assert np.array_equal(y[sample, ..., part], clean[sample, ..., part])


# ------------------------------------------------------------------ log probabilities of tokens

def probs_program(top):
    def f(z, t, *g):
        def split(v):
            outs = nn.token_log_probs(v, t, top)
            return outs[:3], outs[3:]
        outs, pullback, rest = mj.vjp(split, z, has_aux=True)
        return tuple(outs) + tuple(rest) + pullback(tuple(g))
    return f


def check_log_probs(z, t, top):
    rows = t.shape
    g = [normal(11, *rows), normal(12, *rows)] + ([normal(13, *rows, top)] if top else [])
    got, expected, _ = both(probs_program(top), z, t, *g)
    z64, v = z.astype(np.float64).reshape(-1, z.shape[-1]), z.shape[-1]
    with np.errstate(all='ignore'):
        best = np.max(np.where(np.isnan(z64), -np.inf, z64), axis=1)
        best = np.where(np.isfinite(best), best, 0.0)[:, None]
        e = np.where(np.isfinite(z64), np.exp(z64 - best), 0.0)
        s = np.maximum(e.sum(axis=1, keepdims=True), 1e-300)
        spread = np.where(e > 0, np.abs(z64 - best), 0.0)                #|x - max|, rounded once: u of it in the exponent
        mean_spread = (e * spread).sum(axis=1, keepdims=True) / s
        #the sum: every term off by 4 u and by its exponent's rounding (in base 2 the exponent is rounded again, and the
        #factor log2 e itself), then added up
        e_s = (D + 6) * U + 3 * U * mean_spread
        lse = np.abs(best) + np.log(s)
        e_lse = e_s + 4 * U * (np.abs(best) + np.abs(np.log(s)) + 1)
        finite = np.where(np.isfinite(z64), np.abs(z64), 0.0)
        e_lp = e_lse + U * (finite + np.abs(lse)) * 2
        #w / s with w = sum e (x - max): as the sum, with the spread's square mean; and its difference to log s
        mean_square = (e * spread ** 2).sum(axis=1, keepdims=True) / s
        e_h = e_s * (1 + 2 * mean_spread) + ((D + 8) * mean_spread + 3 * mean_square) * U + 8 * U * (np.abs(np.log(s)) + mean_spread + 1)
        p = e / s
        total = sum(np.abs(v.reshape(len(z64), -1)).sum(axis=1, keepdims=True) for v in g)
        logp = np.where(e > 0, np.abs(z64 - best) + np.abs(np.log(s)), 0.0)
        #p = exp(log p): off by log p's error, the exponential's and its exponent's roundings; then the factors
        e_p = p * (e_lp + (3 * logp + 8) * U)
        gh = np.abs(g[1]).reshape(-1, 1)
        entropy = np.abs(np.log(s)) + mean_spread
        e_d = e_p * (total + gh * (logp + entropy)) + p * ((40 + 4) * U * total + gh * (e_lp + e_h + 4 * U * (logp + entropy))) + 8 * U * total
    at = np.where((t.reshape(-1) >= 0) & (t.reshape(-1) < v), t.reshape(-1), 0).astype(np.int64)
    names = ['log_probs', 'entropy'] + (['top'] if top else [])
    bounds = [np.take_along_axis(e_lp, at[:, None], 1)[:, 0], e_h[:, 0]] + ([e_lp.max(axis=1, keepdims=True) * np.ones(top)] if top else [])
    for name, a, b, bound in zip(names, got, expected, bounds):
        close(a.reshape(len(z64), -1), b.reshape(len(z64), -1), np.asarray(bound).reshape(len(z64), -1) + 1e-37, name)
    if top:
        assert np.array_equal(got[3], expected[3])
    close(got[-1].reshape(z64.shape), expected[-1].reshape(z64.shape), e_d + 1e-37, 'gradient')


#(rows, vocabulary): one score, fewer than lanes, odd ones, rows at the edges of vectors, waves and blocks, few rows of many scores
VOCABULARIES = [(1, 1), (3, 2), (130, 10), (5, 63), (67, 64), (9, 65), (70, 255), (300, 256), (9, 257), (33, 1000), (64, 1023), (7, 1024), (5, 1025),
                (6, 2047), (3, 4096), (2, 4099), (5, 8190), (3, 16385), (1, 32000), (2, 50001), (1, 131072), (3, 100003)]


@pytest.mark.parametrize('top', [0, 1, 5, 32])
@pytest.mark.parametrize('rows,v', VOCABULARIES)
def test_log_probs_and_gradient(rows, v, top):
    top = min(top, v)
    print(f'log probabilities {rows} x {v}, top {top}', flush=True)
    rng = np.random.default_rng(rows * v)
    z = normal(1, rows, v, scale=2.5)
    z[:, ::7] = np.round(z[:, ::7])                                       #equal scores
    t = rng.integers(0, v, rows).astype(np.int32)
    if rows > 2:
        t[1], t[rows // 2] = -1, v                                        #padding, below and above
    check_log_probs(z, t, top)


@pytest.mark.parametrize('v', [6, 300, 1028, 5000, 40000])
@pytest.mark.parametrize('order', ['rising', 'falling', 'equal', 'masked', 'late', 'one wave'])
def test_log_probs_of_orders_that_are_hard_for_the_alternatives(order, v):
    print(f'alternatives of {v} scores, {order}', flush=True)
    rng = np.random.default_rng(v)
    z = np.sort(normal(1, 3, v), axis=1)
    if order == 'falling':
        z = np.ascontiguousarray(z[:, ::-1])
    if order == 'equal':
        z[:] = -3.25
        z[1] = -np.inf                                                    #nothing is allowed
        z[2, -2:] = -3.0
    if order == 'masked':
        z[rng.random(z.shape) < 0.9] = -np.inf
        z[0, :-1] = -np.inf
    if order == 'late':
        z = normal(2, 3, v)
        z[:, -40:] += 20.0
    if order == 'one wave':
        #all of the largest in places that one lane, or one wave, reads
        z = normal(2, 3, v)
        z[0, ::64] += 30.0
        z[1, :min(v, 1024)] += 30.0
        z[2, ::256] += 30.0
    check_log_probs(z.astype(f32), np.array([0, v - 1, v // 2], np.int32), min(v, 20))
    check_log_probs(z.astype(f32), np.array([v - 1, 0, -7], np.int32), min(v, 1))


def test_log_probs_of_broken_rows():
    z = normal(1, 6, 700)
    z[0, 5], z[1, 600], z[2, 3], z[2, 699], z[3, :], z[4, 0] = np.nan, np.inf, np.nan, np.inf, np.nan, -np.inf
    check_log_probs(z, np.array([5, 0, 1, 2, 0, -1], np.int32), 4)


@pytest.mark.parametrize('rows,v', [(6, 30000), (1030, 3500), (3, 90001)])
def test_log_probs_of_rows_that_break_late(rows, v):
    z = normal(1, rows, v)
    z[0, v - 100], z[1, v - 2], z[2, v - 1500], z[2, 1] = np.nan, np.inf, np.nan, np.inf
    t = np.arange(rows, dtype=np.int32)
    check_log_probs(z, t, 6)


def test_log_probs_of_scores_far_from_zero():
    z = normal(1, 4, 900)
    z[0] += 3e4
    z[1] -= 3e4
    z[2] *= 50
    z[3, 17] = 3e38
    check_log_probs(z, np.array([1, 2, 3, 17], np.int32), 3)


def test_log_probs_of_unsigned_tokens_and_more_dimensions():
    z = normal(1, 2, 3, 4, 50)
    check_log_probs(z, np.random.default_rng(1).integers(0, 50, (2, 3, 4)).astype(np.int32), 3)
    t = np.random.default_rng(1).integers(0, 50, (2, 3, 4)).astype(np.uint32)
    t[0, 0, 0] = 0xFFFFFFFF
    check_log_probs(z, t, 3)


def test_log_probs_do_not_look_at_padded_rows():
    z = normal(1, 5, 1200)
    z[2], z[4] = np.nan, np.inf
    check_log_probs(z, np.array([3, 4, -1, 5, 1200], np.int32), 2)


# ------------------------------------------------------------------ recurrences

def recurrence_program(gated, reverse, names):
    def f(*arrays):
        a = dict(zip(names, arrays))
        wrt = [n for n in ('factor', 'x', 'state') if n in a]

        def forward(*values):
            d = dict(a, **dict(zip(wrt, values)))
            f = nn.gated_recurrence if gated else lax.linear_recurrence
            return f(d['factor'], d['x'], d.get('state'), d.get('lengths'), reverse)
        outs, pullback = mj.vjp(forward, *[a[n] for n in wrt])
        return tuple(outs) + pullback((a['g'], a['g_last']))
    return f


def check_recurrence(arrays, gated, reverse):
    names = list(arrays)
    got, expected, _ = both(recurrence_program(gated, reverse, names), *arrays.values())
    #One step of the recurrence is off by a few u of its own terms, and carries what came before times a: a recurrence over
    #magnitudes, with a factor that is itself off by 8 u (an exponential, a sum, a division) and joined from parts whose products of
    #factors are each off by as much: 24 u a step covers both, and the last rounding
    a64 = {k: v.astype(np.float64) if v.dtype == f32 else v for k, v in arrays.items()}
    b, t, c = arrays['x'].shape
    inside = np.ones((b, t, c), bool)
    if 'lengths' in arrays:
        inside = np.broadcast_to(np.arange(t)[None, :, None] < arrays['lengths'][:, None, None], inside.shape)
    zero = lambda v: np.where(inside, v, 0.0)
    factor, x = zero(a64['factor']), zero(a64['x'])
    rest = 1 / (1 + np.exp(factor)) if gated else 1.0
    a = np.where(inside, 1 / (1 + np.exp(-factor)) if gated else np.abs(factor), 1.0)
    u = np.abs(zero(rest * x))
    flip = (lambda v: v[:, ::-1]) if reverse else (lambda v: v)

    def walk(a, u, first):
        '''(the recurrence over magnitudes, its error)'''
        size, off = np.abs(first), U * np.abs(first)
        sizes, offs = np.empty_like(u), np.empty_like(u)
        for k in range(t):
            off = a[:, k] * off + 24 * U * (a[:, k] * size + u[:, k])
            size = a[:, k] * size + u[:, k]
            sizes[:, k], offs[:, k] = size, off
        return sizes, offs, size, off
    first = a64.get('state', np.zeros((b, c)))
    sizes, offs, size, off = walk(flip(a), flip(u), first)
    close(got[0], expected[0], flip(offs) + 1e-37, 'h')
    close(got[1], expected[1], off + 1e-37, 'last')
    #the adjoint likewise, from behind
    back = flip(a)[:, ::-1]
    seeds = np.abs(flip(a64['g'])[:, ::-1])
    shifted = np.concatenate([np.ones((b, min(t, 1), c)), back[:, :-1]], axis=1)
    l, e_l, _, _ = walk(shifted, seeds, np.abs(a64['g_last']))
    l, e_l = flip(l[:, ::-1]), flip(e_l[:, ::-1])
    before = flip(np.concatenate([np.abs(first)[:, None], sizes[:, :-1]], axis=1))
    e_before = flip(np.concatenate([U * np.abs(first)[:, None], offs[:, :-1]], axis=1))
    slope = zero(a * rest) if gated else zero(np.ones_like(a))
    inner = before + (np.abs(x) if gated else 0.0)
    close(got[2], expected[2], slope * (e_l * inner + l * e_before + 24 * U * l * inner) + 1e-37, 'dfactor')
    close(got[3], expected[3], zero(rest * np.ones_like(a)) * (e_l + 16 * U * l) + 1e-37, 'dx')
    if 'state' in arrays:
        k = -1 if reverse else 0
        close(got[4], expected[4], a[:, k] * (e_l[:, k] + 16 * U * l[:, k]) + 1e-37, 'dstate')


def recurrence_inputs(b, t, c, gated, state, lengths, seed=0):
    rng = np.random.default_rng(seed)
    arrays = dict(factor=normal(seed + 1, b, t, c, scale=1.5) + f32(2) if gated else (1 - 0.4 * rng.random((b, t, c))).astype(f32), x=normal(seed + 2, b, t, c))
    if state:
        arrays['state'] = normal(seed + 3, b, c)
    if lengths:
        n = rng.integers(0, t + 1, b).astype(np.int32)
        n[:4] = [t, 0, -3, t + 9][:len(n[:4])]
        n[-1] = max(1, t - 1)
        arrays['lengths'] = n
        #what stands behind the ends is not looked at
        behind = np.arange(t)[None, :] >= n[:, None]
        arrays['factor'][behind], arrays['x'][behind] = np.nan, np.inf
    return dict(arrays, g=normal(seed + 4, b, t, c), g_last=normal(seed + 5, b, c))


#(batch, time, channels): single steps, odd ones, times and channels at the edges of chunks and waves, one long sequence, many short ones
RECURRENCES = [(1, 1, 1), (5, 1, 130), (64, 1, 256), (1, 2, 3), (2, 7, 64), (3, 15, 65), (2, 16, 63), (1, 17, 300), (4, 31, 4), (2, 33, 128), (1, 63, 7), (1, 64, 64),
               (2, 65, 68), (1, 127, 1), (1, 128, 192), (2, 257, 100), (1, 511, 33), (1, 1024, 64), (7, 100, 20), (1, 1500, 8), (1, 4097, 5), (70, 9, 12), (3, 640, 260)]


@pytest.mark.parametrize('gated,reverse,state,lengths', [(True, False, True, False), (True, True, True, True), (False, False, False, True), (False, True, True, False),
                                                         (True, False, False, True), (False, False, True, True)])
@pytest.mark.parametrize('b,t,c', RECURRENCES)
def test_recurrence_and_gradient(b, t, c, gated, reverse, state, lengths):
    print(f'recurrence {b} x {t} x {c}, gated {gated}, reverse {reverse}, state {state}, lengths {lengths}', flush=True)
    check_recurrence(recurrence_inputs(b, t, c, gated, state, lengths, seed=b + t + c), gated, reverse)


def test_gates_that_are_open_and_closed():
    arrays = recurrence_inputs(2, 300, 40, True, True, False)
    arrays['factor'][:, ::3] = 200.0                                      #the state stays, to the last bit
    arrays['factor'][:, 1::5] = -200.0                                    #the state is replaced
    arrays['factor'][0, 10], arrays['factor'][1, 20] = np.inf, -np.inf
    with np.errstate(all='ignore'):
        check_recurrence(arrays, True, False)


def test_recurrence_keeps_a_broken_channel_to_itself():
    factor, x = (1 - 0.4 * np.random.default_rng(0).random((2, 200, 70))).astype(f32), normal(1, 2, 200, 70)
    x[0, 50, 3], x[1, 120, 69] = np.nan, np.inf
    f = vkjax_amd.wrap(lambda a, b: lax.linear_recurrence(a, b), frontend='minijax')
    h, last = f(factor, x)
    clean, _ = f(factor, np.where(np.isfinite(x), x, f32(0)))
    ok = np.ones(h.shape, bool)
    ok[0, 50:, 3] = ok[1, 120:, 69] = False
    assert np.array_equal(h[ok], clean[ok]) and np.isnan(h[0, 50:, 3]).all() and not np.isfinite(h[1, 120:, 69]).any()


def test_token_by_token_is_the_whole_run():
    '''A prompt in a padded batch, then single tokens from the state it left.'''
    b, t, c, more = 3, 37, 50, 4
    gate, x = normal(1, b, t + more, c) + f32(1), normal(2, b, t + more, c)
    lengths = np.array([37, 20, 1], np.int32)
    f = vkjax_amd.wrap(lambda *a: nn.gated_recurrence(*a), frontend='minijax')
    _, state = f(gate[:, :t], x[:, :t], np.zeros((b, c), f32), lengths)
    states = [state]
    for k in range(more):
        h, state = f(gate[:, t + k:t + k + 1], x[:, t + k:t + k + 1], state)
        assert np.array_equal(h[:, 0], state)
        states.append(state)
    for i, n in enumerate(lengths):
        pieces = [np.concatenate([v[i:i + 1, :n], v[i:i + 1, t:]], axis=1) for v in (gate, x)]
        whole, _ = f(*pieces, np.zeros((1, c), f32))
        for k, s in enumerate(states):
            #values of at most 5, and 24 u a step of what is kept: a sum of a geometric series of the gates, here below 40
            close(s[i], whole[0, n - 1 + k], 40 * 24 * U * 5)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize('kwargs', [{}, dict(fuse=False), dict(two_lanes=True), dict(graph=True)], ids=['fused', 'unfused', 'lanes', 'graph'])
def test_a_token_models_training_step(kwargs):
    args = token_model_inputs(b=4, t=33, c=32, v=500)
    got, expected, closed = both(token_model_step, *args, **kwargs)
    for a, b in zip(got, expected):
        #products of 32 and 500 terms and three layers: what 32-bit sums of that depth give, relative to the largest value
        assert np.abs(a - b).max() <= 2000 * U * np.abs(b).max(), float(np.abs(a - b).max() / np.abs(b).max())
    again = mj.tree_leaves(vkjax_amd.wrap(token_model_step, frontend='minijax', **kwargs)(*args))
    if kwargs.get('graph'):
        program = JaxprInterpreter(closed, graph=True)
        program.upload_inputs(*args)
        for _ in range(3):
            program.replay(1)
            for k, (a, b) in enumerate(zip(program.read_outputs(), again)):
                #the embedding's gradient is added up by atomics, in any order: a row's sum of at most 132 terms, off by as many u of
                #their magnitudes on either side, which are no larger than the largest value times their number
                table = k == 2 + sorted(args[0]).index('table')
                assert np.array_equal(a.reshape(b.shape), b) or (table and np.abs(a.reshape(b.shape) - b).max() <= 2 * 132 * U * 132 * np.abs(b).max())


def test_operators_give_the_same_bits_every_time():
    f = vkjax_amd.wrap(norm_program(8, 'silu'), frontend='minijax')
    p = vkjax_amd.wrap(probs_program(5), frontend='minijax')
    r = vkjax_amd.wrap(recurrence_program(True, False, ['factor', 'x', 'g', 'g_last']), frontend='minijax')
    norm = [normal(1, 9, 30, 31, 64), normal(2, 64), normal(3, 64), normal(4, 9, 30, 31, 64)]
    z, t = normal(5, 5, 70001), np.array([0, 1, 2, -1, 70000], np.int32)
    probs = [z, t, normal(6, 5), normal(7, 5), normal(8, 5, 5)]
    rec = [v for k, v in recurrence_inputs(1, 5000, 100, True, False, False).items()]
    for g, args in ((f, norm), (p, probs), (r, rec)):
        first = mj.tree_leaves(g(*args))
        for _ in range(3):
            assert all(np.array_equal(a, b) for a, b in zip(first, mj.tree_leaves(g(*args))))
