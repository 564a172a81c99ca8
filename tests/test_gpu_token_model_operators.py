'''Short causal convolutions, selective scans and log probabilities from weights on the GPU against their definitions in 64 bits (the oracle), at the sizes, lengths and
options where they can go wrong.

Tolerances. u = 2^-24 is half a step of fp32. Every multiply-add, product and sum is off by u of its result; a sum of n terms one after the other by at most n u
times the sum of their magnitudes. The sigmoid 1 / (1 + exp2(-z log2 e)) is off by (2 |z| + 6) u of itself (its exponent is rounded twice, the exponential and the
reciprocal are off by at most 2 u each).'''
import numpy as np
import pytest

from tests.test_gpu_operators import U, both, close
from tests.test_operators import normal
from tests.test_token_model_operators import OPTIONAL, loss_program, scan_inputs, scan_program
from oracle import primitives as P
from vkjax_amd import kernels as K, minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

pytestmark = pytest.mark.gpu
jnp, lax, nn = mj.numpy, mj.lax, mj.nn
f32 = np.float32


def inside_of(shape, lengths):
    return np.ones((shape[0], shape[1], 1), bool) if lengths is None else np.arange(shape[1])[None, :, None] < np.clip(np.asarray(lengths), 0, shape[1])[:, None, None]


def spoiled(v, inside):
    '''What stands behind a sequence's end is not to be looked at.'''
    return np.where(inside, v, np.where(np.arange(v.shape[1])[None, :, None] % 2 == 0, np.nan, np.inf)).astype(f32)


# ------------------------------------------------------------------ short causal convolutions

def conv_program(lengths, activation, bias, state):
    def f(x, kernel, g, g_last, *rest):
        given = dict(zip([n for n, has in (('bias', bias), ('state', state)) if has], rest))
        outs, pullback = mj.vjp(lambda x, kernel, given: nn.causal_conv(x, kernel, lengths=lengths, activation=activation, **given), x, kernel, given)
        dx, dkernel, rest = pullback((g, g_last))
        return tuple(outs) + (dx, dkernel) + tuple(rest[n] for n in ('bias', 'state') if n in rest)
    return f


def conv_bounds(x, kernel, g, g_last, bias, state, lengths, activation):
    (batch, time, channels), width = x.shape, kernel.shape[0]
    inside = inside_of(x.shape, lengths)
    front = np.zeros((batch, width - 1, channels)) if state is None else np.abs(state.astype(np.float64))
    rows = np.concatenate([front, np.where(inside, np.abs(x.astype(np.float64)), 0.0)], axis=1)
    k = np.abs(kernel.astype(np.float64))
    size = sum(k[i] * rows[:, i:i + time] for i in range(width)) + (0 if bias is None else np.abs(bias.astype(np.float64)))
    e_z = (width + 1) * U * size
    #silu and its slope: at most 1.1 and |z| + 1 times as large as what they are taken of, slopes at most 1.1 and 0.5
    silu = activation == 'silu'
    e_y = 1.1 * e_z + (2 * size + 10) * U * size if silu else e_z
    e_slope = 0.5 * e_z + (2 * size + 12) * U * (size + 1) if silu else 0 * e_z
    gs = np.where(inside, np.abs(g.astype(np.float64)), 0.0)
    d, e_d = 1.1 * gs, gs * e_slope + 2 * U * gs
    drows, e_drows = np.zeros_like(rows), np.zeros_like(rows)
    n = batch * time                                            #terms of the sums over time
    dkernel = np.zeros(k.shape)
    for i in range(width):
        drows[:, i:i + time] += k[i] * d
        e_drows[:, i:i + time] += k[i] * e_d
        dkernel[i] = (e_d * rows[:, i:i + time] + (n + 2) * U * d * rows[:, i:i + time]).sum(axis=(0, 1))
    for i in range(batch):
        end = time if lengths is None else min(max(int(lengths[i]), 0), time)
        drows[i, end:end + width - 1] += np.abs(g_last[i])
    e_drows += (width + 1) * U * drows
    tiny = 1e-37
    last = np.zeros((batch, width - 1, channels))
    found = [e_y + tiny, last, e_drows[:, width - 1:] + tiny, dkernel + tiny]
    return found + ([(e_d + (n + 1) * U * d).sum(axis=(0, 1)) + tiny] if bias is not None else []) + ([e_drows[:, :width - 1] + tiny] if state is not None else [])


#(shape, width, lengths): one of everything, time shorter than the window, odd channels, more than a tile along time and along channels, steps that are no multiple of a thread's
CONVS = [((1, 1, 1), 2, None), ((2, 1, 64), 4, None), ((2, 1, 64), 4, [0, 1]), ((3, 2, 5), 8, [2, 0, 1]), ((2, 17, 36), 3, [17, 5]), ((1, 300, 8), 4, None), ((4, 33, 130), 5, [33, 32, 2, 0]),
         ((2, 64, 1028), 4, [64, 63]), ((1, 7, 333), 6, [-3]), ((2, 1021, 12), 4, [2000, 700]), ((3, 130, 257), 7, [1, 129, 130]), ((5, 8, 4), 8, [7, 8, 6, 3, 0]), ((1, 5000, 4), 2, None),
         ((40, 9, 32), 4, None)]


@pytest.mark.parametrize('options', [(None, True, True), ('silu', True, False), ('silu', False, True), (None, False, False)], ids=str)
@pytest.mark.parametrize('shape,width,lengths', CONVS, ids=str)
def test_causal_conv_and_gradient(shape, width, lengths, options):
    print(f'causal conv {shape} by {width}, lengths {lengths}, {options}', flush=True)
    activation, has_bias, has_state = options
    inside = inside_of(shape, lengths)
    x, kernel, g = normal(1, *shape), normal(2, width, shape[2]), normal(3, *shape)
    g_last, bias, state = normal(4, shape[0], width - 1, shape[2]), normal(5, shape[2]) if has_bias else None, normal(6, shape[0], width - 1, shape[2]) if has_state else None
    n = None if lengths is None else np.array(lengths, np.int32)
    rest = [v for v in (bias, state) if v is not None]
    got, expected, _ = both(conv_program(n, activation, has_bias, has_state), spoiled(x, inside), kernel, spoiled(g, inside), g_last, *rest)
    names = ['y', 'last', 'dx', 'dkernel'] + ['dbias'] * has_bias + ['dstate'] * has_state
    for name, a, b, bound in zip(names, got, expected, conv_bounds(x, kernel, g, g_last, bias, state, lengths, activation)):
        close(a, b, bound, name)


@pytest.mark.parametrize('width', range(2, 9))
def test_causal_conv_of_every_width(width):
    for shape in ((2, 1, 12), (3, 1, 9), (2, 37, 12), (2, 37, 9)):
        x, kernel, g, g_last, state = (normal(i, *s) for i, s in enumerate((shape, (width, shape[2]), shape, (shape[0], width - 1, shape[2]), (shape[0], width - 1, shape[2]))))
        got, expected, _ = both(conv_program(None, 'silu', False, True), x, kernel, g, g_last, state)
        for k, (a, b, bound) in enumerate(zip(got, expected, conv_bounds(x, kernel, g, g_last, None, state, None, 'silu'))):
            close(a, b, bound, f'{shape}: {k}')


def test_causal_conv_keeps_what_is_not_finite_to_its_window():
    x, kernel = normal(1, 2, 40, 8), normal(2, 4, 8)
    x[0, 10, 3], x[1, 20, 5] = np.nan, np.inf
    got, expected, _ = both(lambda x, k: nn.causal_conv(x, k, activation=None), x, kernel)
    assert np.array_equal(np.isfinite(got[0]), np.isfinite(expected[0])) and (~np.isfinite(got[0])).sum() == 8


# ------------------------------------------------------------------ selective scans

def scan_bounds(v, g, g_last, lengths, softplus):
    '''How far every result of scan_program may be off. Along with the magnitudes H of the states and L of their adjoints (everything positive) goes a bound of their
    errors; a factor exp(w a) is off by what its exponent is (rounded thrice, and w a sum over up to a chunk's steps, T terms) and 2 u.'''
    x, a = v['x'].astype(np.float64), v['a'].astype(np.float64)
    (batch, time, channels), n = x.shape, a.shape[1]
    inside = inside_of(x.shape, lengths)
    clean = lambda w: np.where(inside, w.astype(np.float64), 0.0)
    magnitude = lambda name: np.abs(clean(v[name])) if name in v else None
    pre = clean(v['delta']) + (v['delta_bias'].astype(np.float64) if 'delta_bias' in v else 0.0)
    #delta + bias is rounded; softplus' series, reciprocal, exponential: (|v| + 14) u of itself, and its slope is at most itself (log(1 + e^v) >= sigmoid(v) / 2 for v <= 0.. so 2 times)
    rounded = U * (np.abs(clean(v['delta'])) + (np.abs(v['delta_bias'].astype(np.float64)) if 'delta_bias' in v else 0.0))
    w = np.where(inside, np.maximum(pre, 0) + np.log1p(np.exp(-np.abs(pre))) if softplus else pre, 0.0)
    e_w = np.where(inside, 2 * rounded * np.minimum(w, 1) + (2 * np.abs(pre) + 14) * U * w if softplus else rounded, 0.0)
    xs, bs, cs = np.abs(clean(v['x'])), magnitude('b'), magnitude('c')
    D = np.abs(v['d'].astype(np.float64)) if 'd' in v else 0.0
    open_, e_open, slope = 1.0, 0.0, 0.0
    if 'gate' in v:
        z = clean(v['gate'])
        open_, e_open, slope = np.abs(z / (1 + np.exp(-z))), (2 * np.abs(z) + 10) * U * np.abs(z / (1 + np.exp(-z))), 1.1
    gs = np.abs(clean(g))
    f = np.exp(w[..., None] * a)
    k = f * ((time + 5) * U * np.abs(w[..., None] * a) + e_w[..., None] * np.abs(a) + 2 * U)            #how far a factor is off
    u = w * xs
    e_u = e_w * xs + U * u
    H, E = np.zeros((time + 1, batch, channels, n)), np.zeros((time + 1, batch, channels, n))
    if 'state' in v:
        H[0] = np.abs(v['state'])
    for t in range(time):
        add, e_add = u[:, t, :, None] * bs[:, t, None], e_u[:, t, :, None] * bs[:, t, None]
        H[t + 1] = f[:, t] * H[t] + add
        E[t + 1] = f[:, t] * E[t] + k[:, t] * (H[t] + E[t]) + e_add + 2 * U * add + U * H[t + 1]
        E[t + 1], H[t + 1] = np.where(inside[:, t, :, None], E[t + 1], E[t]), np.where(inside[:, t, :, None], H[t + 1], H[t])
    seen = np.einsum('tbcn,btn->btc', H[1:], cs) + D * xs
    e_seen = np.einsum('tbcn,btn->btc', E[1:], cs) + (n + 3) * U * seen
    e_y = np.where(inside, e_seen * open_ + seen * e_open + 2 * U * seen * open_, 0)
    gy, e_gy = gs * open_, gs * e_open + 2 * U * gs * open_
    #slope of silu: (|z| + 1)(..), off by some (2 |z| + 12) u of (|z| + 1)
    e_dgate = gs * (slope * e_seen + seen * (2 * np.abs(clean(v['gate'])) + 12) * (np.abs(clean(v['gate'])) + 1) * U) if 'gate' in v else None
    L, F = np.abs(g_last.astype(np.float64)), np.zeros((batch, channels, n))
    e_dx, e_dw, e_db, e_dc, e_da, e_dd = np.zeros_like(x), np.zeros_like(x), np.zeros_like(bs), np.zeros_like(cs), np.zeros_like(a), 0.0
    dw = np.zeros_like(x)
    rows = batch * time                                         #terms of sums over time
    absa = np.abs(a)
    for t in range(time - 1, -1, -1):
        add = gy[:, t, :, None] * cs[:, t, None]
        L = L + add
        F = F + e_gy[:, t, :, None] * cs[:, t, None] + U * L
        e_dc[:, t] = (gy[:, t, :, None] * E[t + 1] + e_gy[:, t, :, None] * H[t + 1] + (channels + 2) * U * gy[:, t, :, None] * H[t + 1]).sum(axis=1)
        lb, e_lb = (L * bs[:, t, None]).sum(axis=2), ((F + (n + 1) * U * L) * bs[:, t, None]).sum(axis=2)
        e_db[:, t] = ((F + (channels + 2) * U * L) * u[:, t, :, None] + L * e_u[:, t, :, None]).sum(axis=1)
        back, e_back = f[:, t] * L, f[:, t] * F + k[:, t] * (L + F) + U * f[:, t] * L
        e, e_e = back * H[t], back * E[t] + e_back * (H[t] + E[t]) + U * back * H[t]
        e_da += ((e_e + (rows + 2) * U * e) * w[:, t, :, None] + e * e_w[:, t, :, None]).sum(axis=0)
        dw[:, t] = (e * absa).sum(axis=2) + lb * xs[:, t]
        e_dw[:, t] = ((e_e + (n + 5) * U * e) * absa).sum(axis=2) + e_lb * xs[:, t] + 3 * U * dw[:, t]
        e_dx[:, t] = e_lb * w[:, t] + lb * e_w[:, t] + D * e_gy[:, t] + 3 * U * (lb * w[:, t] + D * gy[:, t])
        L, F = np.where(inside[:, t, :, None], back, L), np.where(inside[:, t, :, None], e_back, F)
    e_ddelta = np.where(inside, e_dw + dw * ((np.abs(pre) + 10) * U + rounded) if softplus else e_dw, 0)
    e_dd = (e_gy * xs + (rows + 2) * U * gy * xs).sum(axis=(0, 1))
    found = dict(x=np.where(inside, e_dx, 0), delta=e_ddelta, a=e_da, b=np.where(inside, e_db, 0), c=np.where(inside, e_dc, 0), d=e_dd,
                 gate=None if e_dgate is None else np.where(inside, e_dgate, 0), state=F + U * L, delta_bias=(e_ddelta + (rows + 2) * U * np.where(inside, dw, 0)).sum(axis=(0, 1)))
    return [b + 1e-36 for b in [e_y, E[time]] + [found[name] for name in v]]


#(batch, time, channels, states, lengths): single steps; states that are no power of two and channels that are no multiple of a wave's; time in chunks (several hundred
#steps), with sequences that end in the first chunk, at its border and behind it; more states than a wave holds
SCANS = [(1, 1, 1, 1, None), (2, 1, 64, 16, None), (3, 1, 5, 7, [0, 1, 1]), (2, 1, 33, 64, None), (1, 2, 3, 4, None), (2, 9, 70, 5, [9, 3]), (1, 130, 64, 16, None), (2, 300, 33, 16, [300, 0]),
         (1, 700, 8, 24, None), (2, 257, 65, 64, [64, 257]), (3, 64, 130, 8, [8, 16, 63]), (1, 1000, 4, 3, None), (4, 40, 200, 2, [40, 1, 39, -5]), (2, 513, 128, 16, [512, 4000]), (1, 129, 1, 33, None),
         (9, 15, 16, 12, None), (1, 300, 33, 8, None)]


@pytest.mark.parametrize('given,softplus', [(OPTIONAL, True), (('gate',), False), (('d', 'state'), True), ((), False), (('delta_bias', 'state'), False)], ids=str)
@pytest.mark.parametrize('batch,time,channels,n,lengths', SCANS, ids=str)
def test_selective_scan_and_gradient(batch, time, channels, n, lengths, given, softplus):
    print(f'selective scan {batch} x {time} x {channels} x {n}, lengths {lengths}, {given}, softplus {softplus}', flush=True)
    arrays, g, g_last = scan_inputs(batch, time, channels, n, given, softplus)
    inside = inside_of((batch, time), lengths)
    dirty = {k: spoiled(v, inside) if k in ('x', 'delta', 'b', 'c', 'gate') else v for k, v in arrays.items()}
    got, expected, _ = both(scan_program(list(arrays), None if lengths is None else np.array(lengths, np.int32), softplus), spoiled(g, inside), g_last, *dirty.values())
    for name, a, b, bound in zip(['y', 'last'] + [f'd{k}' for k in arrays], got, expected, scan_bounds(arrays, g, g_last, lengths, softplus)):
        close(a, b, bound, name)


@pytest.mark.parametrize('batch,time,channels,n,lengths', SCANS, ids=str)
def test_selective_scan_alone(batch, time, channels, n, lengths):
    '''Without a gradient: single steps have a kernel of their own, and no states are kept.'''
    print(f'selective scan {batch} x {time} x {channels} x {n}, lengths {lengths}', flush=True)
    for given, softplus in ((OPTIONAL, True), ((), False)):
        arrays, g, g_last = scan_inputs(batch, time, channels, n, given, softplus, seed=1)
        inside = inside_of((batch, time), lengths)
        dirty = {k: spoiled(v, inside) if k in ('x', 'delta', 'b', 'c', 'gate') else v for k, v in arrays.items()}
        l = None if lengths is None else np.array(lengths, np.int32)
        names = list(arrays)
        got, expected, _ = both(lambda *v: nn.selective_scan(**dict(zip(names, v)), lengths=l, softplus=softplus), *dirty.values())
        for name, a, b, bound in zip(('y', 'last'), got, expected, scan_bounds(arrays, g, g_last, lengths, softplus)):
            close(a, b, bound, name)


@pytest.mark.parametrize('value', [-200.0, -90.0, -30.0, -17.0, -10.0, -1.0, 0.0, 1.0, 20.0, 200.0])
def test_step_widths_far_out(value):
    '''softplus where exp(v) is next to nothing beside 1, and where it is infinite.'''
    arrays, g, g_last = scan_inputs(1, 12, 8, 4, ('state',), True)
    arrays['delta'] = np.full_like(arrays['delta'], value)
    got, expected, _ = both(scan_program(list(arrays), None, True), g, g_last, *arrays.values())
    for name, a, b, bound in zip(['y', 'last'] + [f'd{k}' for k in arrays], got, expected, scan_bounds(arrays, g, g_last, None, True)):
        close(a, b, bound, name)


def test_selective_scan_keeps_what_is_not_finite_to_its_channel():
    arrays, _, _ = scan_inputs(2, 200, 70, 16, (), False)
    arrays['x'][0, 100, 66] = np.nan
    y, last = mj.tree_leaves(both(lambda *v: nn.selective_scan(*v), *arrays.values())[0])
    broken = np.zeros(y.shape, bool)
    broken[0, 100:, 66] = True
    assert np.array_equal(np.isnan(y), broken) and np.isnan(last[0, 66]).all() and np.isfinite(last).sum() == last.size - 16


def test_selective_scan_with_states_that_are_forgotten_at_once():
    #a factor of 0 per step; a sequence's state stays from its length on, which is no multiple of anything here
    for time in (1, 13, 300):
        arrays, _, _ = scan_inputs(3, time, 70, 5, ('state',), False)
        arrays['a'][::7] = -np.inf
        lengths = np.array([time, 0, time // 2], np.int32)
        (y, last), expected, _ = both(lambda *v: nn.selective_scan(**dict(zip(arrays, v)), lengths=lengths), *arrays.values())
        assert np.isfinite(y).all() and np.isfinite(last).all() and np.array_equal(last[1], arrays['state'][1])
        #(one addition, and a sum of five states)
        close(last[:, ::7], expected[1][:, ::7], 4 * U * np.abs(expected[1][:, ::7]) + 1e-37)
        size = 0.2 * np.abs(arrays['x'][:, :, ::7]) * (np.abs(arrays['b']) * np.abs(arrays['c'])).sum(axis=2, keepdims=True)
        close(y[0][:, ::7], expected[0][0][:, ::7], 8 * U * size[0] + 1e-37)


# ------------------------------------------------------------------ log probabilities from weights

def product_error(a, b, terms):
    '''How far a @ b may be off, for magnitudes a and b: operands and products by 12 u of each product (numbers to 2^-22 twice, and what is left out), and by 2^-49 of the operands' largest
    ones; a sum that is rounded twice per 16 terms, and three times where it is put together. (fp32 products are below that.)'''
    return (terms / 8 + 24) * U * (a @ b) + 2.0 ** -49 * terms * a.max(initial=0) * b.max(initial=0)


def loss_bounds(x, w, tokens, g, gs, transposed):
    v64 = w.astype(np.float64).T if transposed else w.astype(np.float64)
    hidden, vocabulary = v64.shape
    given = (tokens >= 0) & (tokens < vocabulary)
    rows = np.where(given[:, None], x.astype(np.float64), 0.0)
    s, e_s = rows @ v64, product_error(np.abs(rows), np.abs(v64), hidden)
    peak = s.max(axis=1, keepdims=True)
    p = np.exp(s - peak)
    p /= p.sum(axis=1, keepdims=True)
    token, at = np.where(given, tokens, 0), np.arange(len(s))
    log_sum = s[at, token] - np.log(p[at, token])
    #exponentials are off by (2 |their argument| + 4) u; the sum of a row's is rounded in a lane (64 times), between lanes and tiles (64 times)
    e_sum = (p * (e_s + (2 * np.abs(s - peak) + 4) * U)).sum(axis=1) + 130 * U
    e_log_sum = e_sum + 4 * U * (np.abs(log_sum) + np.abs(peak[:, 0]))
    e_log_prob = e_log_sum + e_s[at, token] + 4 * U * np.abs(s[at, token])
    of_token, of_sum = np.where(given, g, 0.0).astype(np.float64), np.where(given, gs.astype(np.float64) - g, 0.0)
    #(the largest score and the sum are those of the forward pass: as far off again; q is held to 2^-22 of itself and 2^-49 of its row's larger cotangent)
    relative = e_s + e_s.max(axis=1, keepdims=True) + e_sum[:, None] + (2 * np.abs(s - peak) + 12) * U
    d, e_d = p * np.abs(of_sum)[:, None], p * np.abs(of_sum)[:, None] * relative
    d[at, token] += np.abs(of_token)
    most = np.maximum(np.abs(of_token), np.abs(of_sum))
    e_d += 6 * U * d + 2.0 ** -49 * most[:, None]
    w_abs = np.abs(v64).T
    e_dx = e_d @ w_abs + product_error(d, w_abs, vocabulary)
    e_dw = np.abs(rows).T @ e_d + product_error((np.abs(rows) * most[:, None]).T, d / np.maximum(most, 1e-300)[:, None], len(s))
    tiny = 1e-36
    return [e_log_prob * given + tiny, e_log_sum * given + tiny, e_dx * given[:, None] + tiny, (e_dw.T if transposed else e_dw) + tiny]


def check_loss(x, w, tokens, g, gs, transposed, dirty=None):
    got, expected, _ = both(loss_program(transposed), x if dirty is None else dirty, w, tokens, g, gs)
    for name, a, b, bound in zip(('log_probs', 'log_sums', 'dx', 'dweights'), got, expected, loss_bounds(x, w, tokens, g, gs, transposed)):
        close(a, b, bound, name)


def loss_inputs(rows, hidden, vocabulary, transposed, seed=0):
    rng = np.random.default_rng(seed + rows + 3 * hidden + 7 * vocabulary)
    x, w = rng.standard_normal((rows, hidden)).astype(f32), (rng.standard_normal((hidden, vocabulary)) * 2 / np.sqrt(hidden)).astype(f32)
    tokens = rng.integers(0, vocabulary, rows).astype(np.int32)
    tokens[rng.random(rows) < 0.2] = -1
    tokens[rng.random(rows) < 0.1] = vocabulary
    return x, np.ascontiguousarray(w.T) if transposed else w, tokens, (rng.standard_normal(rows) / rows).astype(f32), (0.1 * rng.standard_normal(rows) / rows).astype(f32)


#(rows, hidden, vocabulary): one of everything; rows that the fp32 instructions take, in one block of 32 and in two, at the border and behind it; contractions of no whole pair of steps; vocabularies that are
#smaller than a vector, end inside a vector, a tile, a block of 32; several tiles each way
LOSSES = [(1, 1, 1), (1, 8, 4), (3, 5, 7), (2, 64, 3), (64, 32, 128), (65, 33, 129), (8, 64, 300), (33, 100, 1001), (130, 70, 515), (257, 128, 4099), (100, 300, 3), (66, 17, 2), (20, 515, 2050),
          (300, 40, 640), (5, 1030, 131), (128, 128, 128), (1100, 9, 1300), (64, 7, 2049), (32, 100, 515), (33, 4, 261), (64, 130, 5000), (7, 3, 50), (17, 257, 6), (1, 300, 9001), (64, 700, 4), (12, 40, 300), (300, 300, 9000), (5, 2100, 131), (40, 1030, 1025), (6, 2050, 17003)]


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('rows,hidden,vocabulary', LOSSES, ids=str)
def test_linear_log_probs_and_gradient(rows, hidden, vocabulary, transposed):
    print(f'linear log probs {rows} x {hidden} x {vocabulary}, transposed {transposed}', flush=True)
    x, w, tokens, g, gs = loss_inputs(rows, hidden, vocabulary, transposed)
    given = (tokens >= 0) & (tokens < vocabulary)
    check_loss(x, w, tokens, g, gs, transposed, np.where(given[:, None], x, np.nan).astype(f32))


@pytest.mark.parametrize('transposed', [False, True])
def test_linear_log_probs_gradient_in_pieces_of_the_vocabulary(transposed, monkeypatch):
    monkeypatch.setattr(K, 'LINEAR_PIECE', 1)
    for rows, hidden, vocabulary in ((140, 70, 600), (40, 130, 513), (520, 33, 300)):
        print(f'in pieces: {rows} x {hidden} x {vocabulary}', flush=True)
        check_loss(*loss_inputs(rows, hidden, vocabulary, transposed), transposed)


def test_linear_log_probs_of_numbers_far_apart():
    '''Rows and columns a thousand times as large as others, and tokens with next to no probability in every row.'''
    x, w, tokens, g, gs = loss_inputs(150, 60, 700, False)
    x *= (10.0 ** np.linspace(-3, 3, 150))[:, None].astype(f32) / 100
    w *= (10.0 ** np.linspace(-4, 0, 700))[None].astype(f32)
    check_loss(x.astype(f32), w.astype(f32), tokens, (g * 1e-6).astype(f32), gs, False)
    x, w, tokens, g, gs = loss_inputs(150, 60, 700, False)
    x[:, 0], w[0] = 1.0, np.linspace(-40, 0, 700)
    check_loss(x, w, tokens, g, gs, False)


@pytest.mark.parametrize('large,small', [(1e33, 1e-33), (1e-33, 1e33), (1e-20, 1e20)])
@pytest.mark.parametrize('rows', [40, 150])
def test_linear_log_probs_of_rows_and_weights_of_different_sizes(rows, large, small):
    x, w, tokens, g, gs = loss_inputs(rows, 60, 700, False)
    x, w = (x * large).astype(f32), (w * small).astype(f32)
    got, expected, _ = both(lambda x, w, t: nn.linear_log_probs(x, w, t), x, w, tokens)
    for name, a, b, bound in zip(('log_probs', 'log_sums'), got, expected, loss_bounds(x, w, tokens, g, gs, False)):
        close(a, b, bound, name)


def test_linear_log_probs_of_one_result_only():
    x, w, tokens, g, _ = loss_inputs(90, 40, 200, False)
    zero = np.zeros_like(g)
    for which in (0, 1):
        f = lambda x, w, tokens, g: mj.vjp(lambda x, w: nn.linear_log_probs(x, w, tokens)[which], x, w)[1](g)
        got, expected, _ = both(f, x, w, tokens, g)
        bounds = loss_bounds(x, w, tokens, *((g, zero) if which == 0 else (zero, g)), False)[2:]
        for name, a, b, bound in zip(('dx', 'dweights'), got, expected, bounds):
            close(a, b, bound, name)


@pytest.mark.parametrize('rows', [9, 200])
def test_linear_log_probs_keep_what_is_not_finite_to_its_row(rows):
    x, w, tokens, g, gs = loss_inputs(rows, 40, 300, False)
    tokens[:] = np.arange(rows) % 300
    x[3, 5], x[6, 0] = np.nan, np.inf
    got = mj.tree_leaves(both(loss_program(False), x, w, tokens, g, gs)[0])
    bad = np.isin(np.arange(rows), (3, 6))
    assert np.array_equal(np.isnan(got[0]), bad) and np.array_equal(np.isnan(got[1]), bad) and np.array_equal(np.isnan(got[2]).all(axis=1), bad) and np.isfinite(got[2][~bad]).all()


def test_linear_log_probs_of_nothing_but_padding():
    for rows in (7, 100):
        x, w, tokens, g, gs = loss_inputs(rows, 40, 300, False)
        got = mj.tree_leaves(both(loss_program(False), np.full_like(x, np.nan), w, np.full_like(tokens, -1), g, gs)[0])
        assert not any(v.any() for v in got)


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('rows', [9, 40, 200])
def test_linear_log_probs_of_weights_that_are_not_finite(rows, transposed):
    x, w, tokens, g, gs = loss_inputs(rows, 40, 300, transposed)
    tokens[::3] = -1
    tokens[1::3] = 5
    w[7, 9] = np.nan
    got = mj.tree_leaves(both(loss_program(transposed), x, w, tokens, g, gs)[0])
    given = (tokens >= 0) & (tokens < 300)
    assert np.array_equal(np.isnan(got[0]), given) and np.array_equal(np.isnan(got[1]), given) and np.isnan(got[2][given]).all()
    assert not any(v[~given].any() for v in got[:3])


# ------------------------------------------------------------------ orthogonalised matrices

def typical_error(a, b):
    '''The root mean square of a product's error, 16 times over: 2^-24 of each term's, terms independent of one another, and what rounding a sum of terms of one sign 64 times leaves.'''
    return 2.0 ** -20 * (np.sqrt((a * a) @ (b * b)) + np.abs(a @ b))


def orthogonal_bound(x, steps, coefficients, eps=1e-7):
    '''How far the result may be off (Frobenius norm). What a step leaves is raised by the steps behind it by no more than the largest difference quotient of their polynomial (of odd
    matrix functions: Daleckii and Krein), the largest slope between 0 and the largest singular value, or value by its argument.'''
    a, b, c = (float(f32(v)) for v in coefficients)
    m = x.astype(np.float64)
    m = m.T if m.shape[0] > m.shape[1] else m
    m = m / (np.sqrt((m * m).sum()) + eps)
    errors, tops = [2.0 ** -21 * np.linalg.norm(m)], []
    for _ in range(steps):
        tops.append(np.linalg.norm(m, 2))
        square = m @ m.T
        e_square = typical_error(m, m.T)
        p = a * np.eye(len(m)) + b * square + c * square @ square
        e_p = abs(b) * e_square + abs(c) * (2 * e_square @ np.abs(square) / np.sqrt(len(m)) + typical_error(square, square)) + 2.0 ** -21 * np.abs(p)
        errors.append(np.linalg.norm(np.sqrt((e_p * e_p) @ (m * m))) + np.linalg.norm(typical_error(p, m)) + 2.0 ** -21 * np.linalg.norm(p @ m))
        m = p @ m
    total = 0.0
    for i, e in enumerate(errors):
        s = np.linspace(1e-9, 1.01 * (tops[i] if i < steps else 1.0), 2000)
        at, slope = s, np.ones_like(s)
        for _ in range(steps - i):
            slope = slope * (a + 3 * b * at**2 + 5 * c * at**4)
            at = a * at + b * at**3 + c * at**5
        total += e * max(np.abs(slope).max(), np.abs(at / s).max())
    return total + 1e-30


#shapes: one element, up to 64 rows either way round (no multiples of 16, one slice of columns and many), fewer rows than a block of 32, wide and tall, no multiples of anything, one tile and several, stacks
MATRICES = [(1, 1), (1, 9), (4, 4), (16, 17), (2, 20, 700), (3, 300, 10), (500, 50), (64, 64), (2, 48, 1000), (64, 5000), (9, 9000), (4097, 63), (40, 64, 20), (5, 3), (2, 7, 40), (33, 65), (128, 128), (3, 130, 100), (2, 2, 64, 200), (257, 129), (300, 520), (20, 32, 31), (129, 1000)]


@pytest.mark.parametrize('steps,coefficients', [(5, (3.4445, -4.7750, 2.0315)), (1, (1.5, -0.5, 0.0)), (2, (2.0, -1.5, 0.5))], ids=str)
@pytest.mark.parametrize('shape', MATRICES, ids=str)
def test_orthogonalize(shape, steps, coefficients):
    print(f'orthogonalize {shape}, {steps} steps, {coefficients}', flush=True)
    x = normal(sum(shape), *shape, scale=1e-3)
    (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x, steps, coefficients), x)
    assert got.shape == shape
    for a, b, m in zip(got.reshape(-1, *shape[-2:]), expected.reshape(-1, *shape[-2:]), x.reshape(-1, *shape[-2:])):
        off, bound = np.linalg.norm(a.astype(np.float64) - b), orthogonal_bound(m, steps, coefficients)
        assert off <= bound, (off, bound)


@pytest.mark.parametrize('scale', [1e-12, 1e-7, 1e15])
def test_orthogonalize_by_the_size_of_its_matrix(scale):
    x = normal(1, 40, 50, scale=scale)
    (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x), x)
    assert np.linalg.norm(got.astype(np.float64) - expected) <= orthogonal_bound(x, 5, (3.4445, -4.7750, 2.0315))


@pytest.mark.parametrize('rows,columns', [(150, 90), (40, 90), (300, 64)])
def test_orthogonalize_a_matrix_of_a_low_rank_and_of_zeros(rows, columns):
    x = normal(1, 4, rows, columns, scale=1e-2)
    x[1] = normal(2, rows, 2) @ normal(3, 2, columns)
    x[2] = 0.0
    x[3, 7, 8] = np.nan
    (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x), x)
    assert not got[2].any() and np.isnan(got[3]).all()
    for i in (0, 1):
        assert np.linalg.norm(got[i].astype(np.float64) - expected[i]) <= orthogonal_bound(x[i], 5, (3.4445, -4.7750, 2.0315))


@pytest.mark.parametrize('steps', [1, 5, 6, 7, 18, 32])
def test_orthogonalize_singular_values_far_apart(steps):
    #a few rows, of which the smallest singular values are 1e-4 of the largest: what the squares of those lose in fp32 would decide where they go
    for coefficients in ((3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0)):
        u, _, v = np.linalg.svd(normal(7, 30, 400), full_matrices=False)
        x = (u * np.logspace(0, -4, 30) @ v).astype(f32)
        (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x, steps, coefficients), x)
        off, bound = np.linalg.norm(got.astype(np.float64) - expected), orthogonal_bound(x, steps, coefficients)
        assert off <= bound, (off, bound)


@pytest.mark.parametrize('rows', [9, 64, 150])
def test_gradient_of_log_probs_with_and_without_what_was_kept(rows):
    x, w, tokens, g, gs = loss_inputs(rows, 70, 600, False)

    def both_ways(x, w, tokens, g, gs):
        outs = lax.linear_log_probs(x, w, tokens, with_parts=True)
        return lax.linear_log_probs_grad(x, w, tokens, outs[2], outs[3], g, gs, parts=outs[4:]) + lax.linear_log_probs_grad(x, w, tokens, outs[2], outs[3], g, gs)
    (dx, dw, dx2, dw2), _, _ = both(both_ways, x, w, tokens, g, gs)
    assert np.array_equal(dx, dx2) and np.array_equal(dw, dw2)


# ------------------------------------------------------------------ products whose contraction is shared

@pytest.mark.parametrize('slices', [1, 2, 5, 40])
@pytest.mark.parametrize('kernel,side', [(k[0], k[1]) for k in K.HALF_KERNELS])
def test_products_that_share_contractions(kernel, side, slices, monkeypatch):
    '''Several hundred blocks that leave parts of sums for one another: every kernel, some tiles by one block and the others shared, more slices than pairs of steps among them. The result does not
    depend on who comes last.'''
    print(f'shared contractions: {kernel}, {slices} slices', flush=True)
    #(tiles of 64 that run two to a CU share the contraction of 1300 alone)
    chosen = lambda pairs: '_64_many' if kernel == '_64' and slices > 1 and pairs != 41 else kernel
    monkeypatch.setattr(K, 'half_plan', lambda tiles_of, pairs: K.HalfPlan(chosen(pairs), side, 0 if slices > 1 else tiles_of(side), min(slices, pairs)))
    x = normal(1, 1100, 1300)
    f = mj.make_jaxpr(lambda x: nn.orthogonalize(x, 1))(x)
    program = JaxprInterpreter(f)
    first, = program.run(x)
    off = np.linalg.norm(first.astype(np.float64) - P.orthogonalize(x, 1, (3.4445, -4.7750, 2.0315), 1e-7))
    assert off <= orthogonal_bound(x, 1, (3.4445, -4.7750, 2.0315)), off
    for _ in range(4):
        assert np.array_equal(program.run(x)[0], first)
    y = normal(2, 1100, 1300)
    other, = program.run(y)
    assert np.linalg.norm(other.astype(np.float64) - P.orthogonalize(y, 1, (3.4445, -4.7750, 2.0315), 1e-7)) <= orthogonal_bound(y, 1, (3.4445, -4.7750, 2.0315))
    assert np.array_equal(program.run(x)[0], first)


def test_gradient_of_log_probs_with_shared_contractions(monkeypatch):
    x, w, tokens, g, gs = loss_inputs(700, 300, 1500, False)
    for kernel, side, *_ in K.HALF_KERNELS:
        for slices in (1, 3):
            print(f'gradient with shared contractions: {kernel}, {slices} slices', flush=True)
            monkeypatch.setattr(K, 'half_plan', lambda tiles_of, pairs: K.HalfPlan(kernel, side, 3 if slices > 1 else tiles_of(side), min(slices, pairs)))
            check_loss(x, w, tokens, g, gs, False)


@pytest.mark.parametrize('n,rows,columns,steps', [(700, 20, 30, 1), (700, 20, 30, 3), (600, 64, 66, 5), (1100, 12, 9, 2)])
def test_orthogonalize_many_matrices(n, rows, columns, steps):
    x = normal(n, n, rows, columns)
    (got,), (expected,), _ = both(lambda x: nn.orthogonalize(x, steps), x)
    for i in (0, 1, n // 2, n - 2, n - 1):
        off, bound = np.linalg.norm(got[i].astype(np.float64) - expected[i]), orthogonal_bound(x[i], steps, (3.4445, -4.7750, 2.0315))
        assert off <= bound, (i, off, bound)
    assert np.isfinite(got).all() and (np.linalg.norm(got - expected, axis=(1, 2)) < 0.05 * np.sqrt(min(rows, columns))).all()
