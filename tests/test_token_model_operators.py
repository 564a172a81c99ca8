'''Operators of a recurrent token model as programs: what they and their gradients are (the oracle against torch in 64 bits and against
differences), what is refused, and how they are planned.'''
import numpy as np
import pytest
import torch

from oracle import primitives as P
from tests.test_operators import ROUNDED, evaluate, normal, refused
from vkjax_amd import kernels as K, minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

jnp, lax, nn = mj.numpy, mj.lax, mj.nn
f32 = np.float32


def leaf(v):
    return None if v is None else torch.tensor(np.asarray(v, np.float64), requires_grad=True)


def same_as_torch(got, expected):
    for a, b in zip(got, expected):
        assert np.allclose(a, b.detach().numpy(), **dict(ROUNDED, atol=1e-12)), float(np.abs(a - b.detach().numpy()).max())


# ------------------------------------------------------------------ short causal convolutions

def torch_conv(x, kernel, bias, state, ends, silu):
    '''One sequence after the other, position by position.'''
    ys, lasts = [], []
    width = kernel.shape[0]
    for i, n in enumerate(ends):
        front = torch.zeros(width - 1, x.shape[2], dtype=x.dtype) if state is None else state[i]
        rows = torch.cat([front, x[i, :n]])
        out = [(kernel * rows[t:t + width]).sum(0) + (0 if bias is None else bias) for t in range(n)]
        y = torch.stack(out) if out else x[i, :0]
        ys.append(torch.cat([torch.nn.functional.silu(y) if silu else y, torch.zeros_like(x[i, n:])]))
        lasts.append(rows[n:])
    return torch.stack(ys), torch.stack(lasts)


@pytest.mark.parametrize('activation', [None, 'silu'])
@pytest.mark.parametrize('width,shape,bias,state,lengths', [(2, (2, 5, 3), True, True, None), (4, (3, 6, 2), True, False, [6, 0, 2]), (8, (2, 3, 4), False, True, [1, 3]),
                                                            (3, (1, 1, 1), False, False, None), (4, (2, 1, 3), True, True, [0, 1])])
def test_causal_conv_oracle_is_torchs(width, shape, bias, state, lengths, activation):
    x, kernel, g, g_last = normal(1, *shape), normal(2, width, shape[2]), normal(3, *shape), normal(4, shape[0], width - 1, shape[2])
    b, s = normal(5, shape[2]) if bias else None, normal(6, *g_last.shape) if state else None
    ends = [shape[1]] * shape[0] if lengths is None else lengths
    n = None if lengths is None else np.array(lengths, np.int32)

    def f(x, kernel, *rest):
        rest = list(rest)
        given = dict(bias=rest.pop(0) if bias else None, state=rest.pop(0) if state else None)
        outs, pullback = mj.vjp(lambda x, kernel, given: nn.causal_conv(x, kernel, lengths=n, activation=activation, **given), x, kernel, given)
        dx, dkernel, rest = pullback((g, g_last))
        return tuple(outs) + (dx, dkernel) + tuple(v for v in (rest['bias'], rest['state']) if v is not None)
    got = evaluate(f, x, kernel, *[v for v in (b, s) if v is not None])
    leaves = [leaf(v) for v in (x, kernel, b, s)]
    y, last = torch_conv(*leaves, ends, activation == 'silu')
    ((y * torch.tensor(g)).sum() + (last * torch.tensor(g_last)).sum()).backward()
    same_as_torch(got, [y, last] + [v.grad for v in leaves if v is not None])


def test_causal_conv_goes_on_token_by_token():
    x, kernel, bias = normal(1, 2, 7, 3), normal(2, 4, 3), normal(3, 3)

    def whole(x, kernel, bias):
        return nn.causal_conv(x, kernel, bias, activation='silu')

    def steps(x, kernel, bias):
        state, ys = None, []
        for t in range(7):
            y, state = nn.causal_conv(x[:, t:t + 1], kernel, bias, state, activation='silu')
            ys.append(y)
        return jnp.concatenate(ys, axis=1), state
    for a, b in zip(evaluate(whole, x, kernel, bias), evaluate(steps, x, kernel, bias)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize('change,error', [
    (dict(x=np.ones((2, 12), f32)), TypeError), (dict(x=np.ones((2, 3, 4), np.int32)), TypeError), (dict(kernel=np.ones((4, 5), f32)), TypeError),
    (dict(kernel=np.ones((1, 4), f32)), ValueError), (dict(kernel=np.ones((9, 4), f32)), ValueError), (dict(kernel=np.ones((3, 4), f32)), TypeError),
    (dict(bias=np.ones(3, f32)), TypeError), (dict(state=np.ones((2, 4, 4), f32)), TypeError), (dict(state=np.ones((2, 3, 4), np.int32)), TypeError),
    (dict(lengths=np.ones(3, np.int32)), TypeError), (dict(lengths=np.ones(2, f32)), TypeError), (dict(activation='relu'), ValueError)])
def test_causal_conv_refuses(change, error):
    given = dict(dict(x=np.ones((2, 3, 4), f32), kernel=np.ones((4, 4), f32), bias=np.ones(4, f32), state=np.ones((2, 3, 4), f32), lengths=np.ones(2, np.int32), activation='silu'), **change)
    activation = given.pop('activation')
    refused(error, lambda *a: nn.causal_conv(*a, activation), *given.values())
    refused(error, lambda *a: lax.causal_conv_grad(*a, None, None, activation), *given.values())


def test_causal_conv_gradient_refuses_cotangents_of_other_shapes():
    x, kernel = np.ones((2, 3, 4), f32), np.ones((4, 4), f32)
    refused(TypeError, lambda x, k, g: lax.causal_conv_grad(x, k, g=g), x, kernel, np.ones((2, 4, 4), f32))
    refused(TypeError, lambda x, k, g: lax.causal_conv_grad(x, k, g_last=g), x, kernel, x.repeat(2, 1))


# ------------------------------------------------------------------ selective scans

def torch_scan(x, delta, a, b, c, d, gate, state, bias, ends, softplus):
    ys, lasts = [], []
    for i, n in enumerate(ends):
        h = torch.zeros(a.shape, dtype=a.dtype) if state is None else state[i]
        out = []
        for t in range(n):
            w = delta[i, t] if bias is None else delta[i, t] + bias
            w = torch.nn.functional.softplus(w, threshold=1e9) if softplus else w
            h = torch.exp(w[:, None] * a) * h + (w * x[i, t])[:, None] * b[i, t]
            y = h @ c[i, t]
            y = y if d is None else y + d * x[i, t]
            out.append(y if gate is None else y * torch.nn.functional.silu(gate[i, t]))
        ys.append(torch.cat([torch.stack(out), torch.zeros_like(x[i, n:])]) if out else torch.zeros_like(x[i]))
        lasts.append(h + 0)
    return torch.stack(ys), torch.stack(lasts)


OPTIONAL = ('d', 'gate', 'state', 'delta_bias')


def scan_inputs(batch, time, channels, n, given, softplus, seed=0):
    '''Operands as a model has them: step widths around 0.05, states that decay.'''
    rng = np.random.default_rng(seed + 7 * time + channels)
    draw = lambda *s: rng.standard_normal(s).astype(f32)
    found = dict(x=draw(batch, time, channels),
                 delta=(0.7 * draw(batch, time, channels) - (0.0 if 'delta_bias' in given else 3.0)).astype(f32) if softplus else (0.01 + 0.1 * rng.random((batch, time, channels))).astype(f32),
                 a=(-(0.5 + rng.random((channels, n))) * np.arange(1, n + 1)).astype(f32), b=draw(batch, time, n), c=draw(batch, time, n))
    shapes = dict(d=(channels,), gate=(batch, time, channels), state=(batch, channels, n), delta_bias=(channels,))
    found.update({name: draw(*shapes[name]) for name in OPTIONAL if name in given})
    if 'delta_bias' in given:
        found['delta_bias'] = (found['delta_bias'] - 3.0).astype(f32) if softplus else (0.01 * rng.random(channels)).astype(f32)
    return found, draw(batch, time, channels), draw(batch, channels, n)


def scan_program(names, lengths, softplus):
    '''Results and gradients of every operand, in the order of `names`.'''
    def f(g, g_last, *arrays):
        outs, pullback = mj.vjp(lambda *v: nn.selective_scan(**dict(zip(names, v)), lengths=lengths, softplus=softplus), *arrays)
        return tuple(outs) + pullback((g, g_last))
    return f


@pytest.mark.parametrize('softplus', [False, True])
@pytest.mark.parametrize('batch,time,channels,n,given,lengths', [(2, 5, 3, 4, OPTIONAL, None), (3, 6, 2, 1, ('gate',), [6, 0, 2]), (1, 1, 4, 16, ('state', 'delta_bias'), None),
                                                                 (2, 17, 3, 5, ('d', 'state'), [17, 9]), (2, 9, 1, 3, (), None)])
def test_selective_scan_oracle_is_torchs(batch, time, channels, n, given, lengths, softplus):
    arrays, g, g_last = scan_inputs(batch, time, channels, n, given, softplus)
    got = evaluate(scan_program(list(arrays), None if lengths is None else np.array(lengths, np.int32), softplus), g, g_last, *arrays.values())
    leaves = {k: leaf(v) for k, v in arrays.items()}
    y, last = torch_scan(*[leaves[k] for k in ('x', 'delta', 'a', 'b', 'c')], *[leaves.get(k) for k in OPTIONAL], [time] * batch if lengths is None else lengths, softplus)
    ((y * torch.tensor(g)).sum() + (last * torch.tensor(g_last)).sum()).backward()
    grad = lambda v: torch.zeros_like(v) if v.grad is None else v.grad
    same_as_torch(got, [y, last] + [grad(v) for v in leaves.values()])


def test_selective_scan_gradient_is_that_of_differences():
    arrays, g, g_last = scan_inputs(2, 4, 2, 3, OPTIONAL, True)
    names = list(arrays)
    flags = dict(softplus=True, has_d=True, has_gate=True, has_state=True, has_lengths=False, has_bias=True)

    def loss(values):
        _, inside, _, _, _, _, _, _, h, seen, open_, _ = P._selective_scan64(*[values[k] for k in ('x', 'delta', 'a', 'b', 'c', 'd', 'gate', 'state')], None, values['delta_bias'], True)
        return (seen * open_ * g).sum() + (h[-1] * g_last).sum()
    wide = {k: v.astype(np.float64) for k, v in arrays.items()}
    grads = dict(zip(names, P.selective_scan_grad(None, *arrays.values(), g, g_last, has_g=True, has_last=True, **flags)))
    for name in names:
        for at in np.ndindex(*wide[name].shape):
            ends = []
            for step in (1e-5, -1e-5):
                moved = dict(wide, **{name: wide[name].copy()})
                moved[name][at] += step
                ends.append(loss(moved))
            assert abs((ends[0] - ends[1]) / 2e-5 - grads[name][at]) < 2e-5 * max(1.0, abs(grads[name][at])), (name, at)


def test_selective_scan_goes_on_in_pieces():
    arrays, _, _ = scan_inputs(2, 9, 3, 4, ('d', 'gate', 'delta_bias'), True)
    per_step = ('x', 'delta', 'b', 'c', 'gate')

    def whole(arrays):
        return nn.selective_scan(**arrays, softplus=True)

    def pieces(arrays):
        state, ys = None, []
        for lo, hi in ((0, 5), (5, 6), (6, 6), (6, 9)):
            y, state = nn.selective_scan(**{k: v[:, lo:hi] if k in per_step else v for k, v in arrays.items()}, state=state, softplus=True)
            ys.append(y)
        return jnp.concatenate(ys, axis=1), state
    #(the state is rounded to fp32 between pieces)
    for a, b in zip(evaluate(whole, arrays), evaluate(pieces, arrays)):
        assert np.allclose(a, b, rtol=1e-5, atol=1e-6)


BAD_SCANS = [(dict(x=np.ones((2, 12), f32)), TypeError), (dict(x=np.ones((2, 3, 4), np.int32)), TypeError), (dict(delta=np.ones((2, 3, 5), f32)), TypeError),
             (dict(a=np.ones((5, 6), f32)), TypeError), (dict(a=np.ones((4, 65), f32), b=np.ones((2, 3, 65), f32), c=np.ones((2, 3, 65), f32), state=np.ones((2, 4, 65), f32)), ValueError),
             (dict(a=np.ones((4, 0), f32)), ValueError), (dict(b=np.ones((2, 3, 5), f32)), TypeError), (dict(c=np.ones((2, 4, 6), f32)), TypeError), (dict(d=np.ones(3, f32)), TypeError),
             (dict(gate=np.ones((2, 3, 1), f32)), TypeError), (dict(state=np.ones((2, 6, 4), f32)), TypeError), (dict(lengths=np.ones(2, f32)), TypeError),
             (dict(lengths=np.ones((2, 1), np.int32)), TypeError), (dict(delta_bias=np.ones((1, 4), f32)), TypeError), (dict(delta=np.ones((2, 3, 4), bool)), TypeError)]


@pytest.mark.parametrize('change,error', BAD_SCANS)
def test_selective_scan_refuses(change, error):
    given = dict(dict(x=np.ones((2, 3, 4), f32), delta=np.ones((2, 3, 4), f32), a=np.ones((4, 6), f32), b=np.ones((2, 3, 6), f32), c=np.ones((2, 3, 6), f32), d=np.ones(4, f32),
                      gate=np.ones((2, 3, 4), f32), state=np.ones((2, 4, 6), f32), lengths=np.ones(2, np.int32), delta_bias=np.ones(4, f32)), **change)
    refused(error, lambda *a: nn.selective_scan(*a), *given.values())
    refused(error, lambda *a: lax.selective_scan_grad(np.ones((1, 2, 6, 4), f32), *a), *given.values())


def test_selective_scan_gradient_refuses_what_does_not_belong():
    x, a, b = np.ones((2, 9, 4), f32), np.ones((4, 6), f32), np.ones((2, 9, 6), f32)
    kept = np.ones((2, 2, 6, 4), f32)
    refused(TypeError, lambda *v: lax.selective_scan_grad(*v), kept[:1], x, x, a, b, b)
    refused(TypeError, lambda *v: lax.selective_scan_grad(*v[:6], g=v[6]), kept, x, x, a, b, b, b)
    refused(TypeError, lambda *v: lax.selective_scan_grad(*v[:6], g_last=v[6]), kept, x, x, a, b, b, np.ones((2, 6, 4), f32))
    refused(NotImplementedError, lambda *v: mj.vjp(lambda x: lax.selective_scan(x, *v[1:], with_kept=True)[2], x)[1](kept), x, x, a, b, b)


# ------------------------------------------------------------------ planning

@pytest.mark.parametrize('shape', [(0, 5, 4), (3, 0, 4), (3, 5, 0)])
def test_arrays_without_elements_are_planned(shape):
    batch, time, channels = shape
    x, kernel, state, g_last = np.zeros(shape, f32), normal(1, 4, channels), normal(2, batch, 3, channels), normal(3, batch, 3, channels)

    def conv(x, kernel, state, g_last):
        outs, pullback = mj.vjp(lambda x, k, s: nn.causal_conv(x, k, None, s), x, kernel, state)
        return tuple(outs) + pullback((x, g_last))
    y, last, dx, dkernel, dstate = evaluate(conv, x, kernel, state, g_last)
    assert np.array_equal(last, state) and np.array_equal(dstate, g_last) and y.shape == dx.shape == shape and not dkernel.any()
    JaxprInterpreter(mj.make_jaxpr(conv)(x, kernel, state, g_last), plan_only=True)
    arrays, g, g_last = scan_inputs(batch, time, channels, 3, OPTIONAL, True)
    f = scan_program(list(arrays), None, True)
    outs = evaluate(f, g, g_last, *arrays.values())
    assert np.array_equal(outs[1], arrays['state']) and not outs[4].any() and np.array_equal(outs[2 + list(arrays).index('state')], g_last)
    JaxprInterpreter(mj.make_jaxpr(f)(g, g_last, *arrays.values()), plan_only=True)


def test_the_states_that_a_gradient_needs_are_kept_only_then():
    arrays, g, g_last = scan_inputs(1, 40, 8, 4, (), False)
    names = list(arrays)
    kept = lambda program: [e.params['kept'] for e in mj.make_jaxpr(program)(g, g_last, *arrays.values()).jaxpr.eqns if e.primitive.name == 'selective_scan']
    assert kept(lambda g, last, *v: nn.selective_scan(**dict(zip(names, v)))) == [False]
    assert kept(scan_program(names, None, False)) == [True]


# ------------------------------------------------------------------ log probabilities from weights

def loss_program(transposed):
    def f(x, weights, tokens, g_log_probs, g_log_sums):
        outs, pullback = mj.vjp(lambda x, w: nn.linear_log_probs(x, w, tokens, transposed), x, weights)
        return tuple(outs) + pullback((g_log_probs, g_log_sums))
    return f


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('shape,hidden,vocabulary', [((5,), 7, 11), ((2, 3), 4, 6), ((), 3, 5), ((4,), 1, 1)])
def test_linear_log_probs_oracle_is_torchs(shape, hidden, vocabulary, transposed):
    x, w = normal(1, *shape, hidden), normal(2, *((vocabulary, hidden) if transposed else (hidden, vocabulary)))
    tokens = np.random.default_rng(3).integers(-1, vocabulary + 1, shape).astype(np.int32)
    g, gs = normal(4, *shape) if shape else f32(0.7), normal(5, *shape) if shape else f32(-0.2)
    got = evaluate(loss_program(transposed), x, w, tokens, g, gs)
    tx, tw = leaf(x), leaf(w)
    scores = tx @ (tw.T if transposed else tw)
    token  = torch.tensor(np.asarray(tokens, np.int64))
    given  = (token >= 0) & (token < vocabulary)
    log_sum = torch.where(given, torch.logsumexp(scores, -1), 0.0)
    log_prob = torch.where(given, torch.gather(torch.log_softmax(scores, -1), -1, token.clamp(0, vocabulary - 1)[..., None])[..., 0], 0.0)
    ((log_prob * torch.tensor(g)).sum() + (log_sum * torch.tensor(gs)).sum()).backward()
    same_as_torch(got, [log_prob, log_sum, tx.grad, tw.grad])


def test_linear_log_probs_are_the_log_probs_of_the_product():
    x, w, tokens = normal(1, 6, 5), normal(2, 5, 9), np.array([0, 8, -1, 3, 9, 3], np.int32)
    a = evaluate(lambda x, w: nn.linear_log_probs(x, w, tokens)[0], x, w)[0]
    b = evaluate(lambda x, w: nn.token_log_probs(jnp.dot(x, w), tokens)[0], x, w)[0]
    assert np.allclose(a, b, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize('change,error', [
    (dict(x=np.ones((3, 5), f32)), TypeError), (dict(x=np.ones((3, 4), np.int32)), TypeError), (dict(weights=np.ones((7, 4), f32)), TypeError), (dict(weights=np.ones(4, f32)), TypeError),
    (dict(weights=np.ones((4, 0), f32)), TypeError), (dict(x=np.ones((3, 0), f32), weights=np.ones((0, 7), f32)), TypeError), (dict(tokens=np.ones(4, np.int32)), TypeError),
    (dict(tokens=np.ones((3, 1), np.int32)), TypeError), (dict(tokens=np.ones(3, f32)), TypeError), (dict(x=np.ones((), f32), tokens=np.ones((), np.int32)), TypeError)])
def test_linear_log_probs_refuse(change, error):
    given = dict(dict(x=np.ones((3, 4), f32), weights=np.ones((4, 7), f32), tokens=np.ones(3, np.int32)), **change)
    refused(error, lambda *a: nn.linear_log_probs(*a), *given.values())
    refused(error, lambda *a: lax.linear_log_probs_grad(*a, np.ones(3, f32), np.ones(3, f32)), *given.values())


def test_linear_log_probs_refuse_weights_the_other_way_round():
    x, t = np.ones((3, 4), f32), np.ones(3, np.int32)
    refused(TypeError, lambda x, w, t: nn.linear_log_probs(x, w, t, transposed=True), x, np.ones((4, 7), f32), t)
    refused(TypeError, lambda x, w, t: nn.linear_log_probs(x, w, t), x, np.ones((7, 4), f32), t)


def test_linear_log_probs_gradient_refuses_what_does_not_belong():
    x, w, t, row = np.ones((3, 4), f32), np.ones((4, 7), f32), np.ones(3, np.int32), np.ones(3, f32)
    for bad in (np.ones(4, f32), np.ones((3, 1), f32), np.ones(3, np.int32)):
        for at in range(4):
            values = [row] * 4
            values[at] = bad
            refused(TypeError, lambda *a: lax.linear_log_probs_grad(*a), x, w, t, *values)
    refused(NotImplementedError, lambda x, w, t, g: mj.vjp(lambda x: lax.linear_log_probs(x, w, t)[2], x)[1](g), x, w, t, row)


def test_log_probs_of_no_rows_are_planned():
    x, w, t, g = np.zeros((0, 4), f32), normal(1, 4, 7), np.zeros(0, np.int32), np.zeros(0, f32)
    _, _, dx, dw = evaluate(loss_program(False), x, w, t, g, g)
    assert dx.shape == (0, 4) and not dw.any()
    JaxprInterpreter(mj.make_jaxpr(loss_program(False))(x, w, t, g, g), plan_only=True)


# ------------------------------------------------------------------ orthogonalised matrices

@pytest.mark.parametrize('shape', [(4, 7), (7, 4), (2, 3, 5, 5), (1, 1), (1, 6)])
@pytest.mark.parametrize('steps,coefficients', [(5, (3.4445, -4.7750, 2.0315)), (1, (2.0, -1.5, 0.5)), (20, (1.5, -0.5, 0.0))])
def test_orthogonalize_is_a_polynomial_of_the_singular_values(shape, steps, coefficients):
    x = normal(1, *shape)
    got, = evaluate(lambda x: nn.orthogonalize(x, steps, coefficients), x)
    a, b, c = (float(f32(v)) for v in coefficients)
    u, s, v = np.linalg.svd(x.astype(np.float64), full_matrices=False)
    s = s / (np.sqrt((x.astype(np.float64) ** 2).sum(axis=(-2, -1), keepdims=True))[..., 0] + float(f32(1e-7)))
    for _ in range(steps):
        s = a * s + b * s**3 + c * s**5
    #(64 bits, whose roundings the steps raise by 3.5^5 at most, then one to fp32 of values below 2)
    assert np.allclose(got, u @ (s[..., None] * v), rtol=0, atol=1e-10 + 2.0 ** -23)


def test_orthogonalize_brings_singular_values_to_one():
    for shape in ((20, 30), (30, 20)):
        s = np.linalg.svd(evaluate(lambda x: nn.orthogonalize(x), normal(2, *shape))[0], compute_uv=False)
        assert s.min() > 0.6 and s.max() < 1.3
        s = np.linalg.svd(evaluate(lambda x: nn.orthogonalize(x, 25, (1.5, -0.5, 0.0)), normal(2, *shape))[0], compute_uv=False)
        assert np.allclose(s, 1.0, atol=1e-5)


def test_orthogonalize_of_zeros_and_of_matrices_by_themselves():
    x = normal(1, 3, 4, 6)
    x[0], x[1, 2, 3] = 0.0, np.nan
    got, = evaluate(lambda x: nn.orthogonalize(x), x)
    alone, = evaluate(lambda x: nn.orthogonalize(x), x[2])
    assert not got[0].any() and np.isnan(got[1]).all() and np.array_equal(got[2], alone)


@pytest.mark.parametrize('change,error', [
    (dict(x=np.ones(4, f32)), TypeError), (dict(x=np.ones((4, 4), np.int32)), TypeError), (dict(steps=0), ValueError), (dict(steps=33), ValueError), (dict(steps=2.5), ValueError),
    (dict(coefficients=(1.0, 2.0)), ValueError), (dict(coefficients=(1.0, np.nan, 0.0)), ValueError), (dict(coefficients=(3.0, 2.0, 1.0)), ValueError), (dict(eps=0.0), ValueError),
    (dict(eps=-1e-7), ValueError), (dict(eps=np.inf), ValueError)])
def test_orthogonalize_refuses(change, error):
    given = dict(dict(x=np.ones((4, 4), f32), steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7), **change)
    refused(error, lambda x: nn.orthogonalize(x, given['steps'], given['coefficients'], given['eps']), given['x'])


def test_orthogonalize_has_no_gradient_and_takes_no_elements():
    refused(NotImplementedError, lambda x: mj.grad(lambda v: jnp.sum(nn.orthogonalize(v)))(x), np.ones((3, 4), f32))
    for shape in ((0, 4), (4, 0), (0, 3, 4)):
        assert evaluate(lambda x: nn.orthogonalize(x), np.zeros(shape, f32))[0].shape == shape
        JaxprInterpreter(mj.make_jaxpr(lambda x: nn.orthogonalize(x))(np.zeros(shape, f32)), plan_only=True)


def test_orthogonalize_knows_how_large_singular_values_become():
    rng = np.random.default_rng(0)
    for steps, coefficients in ((5, (3.4445, -4.7750, 2.0315)), (8, (3.4445, -4.7750, 2.0315)), (6, (1.5, -0.5, 0.0)), (4, (2.0, -1.5, 0.5)), (3, (1.0, 0.5, 0.25))):
        a, b, c = coefficients
        s = rng.random(200000)
        for most, polynomial in K.orthogonal_bounds(steps, coefficients):
            p = a + b * s**2 + c * s**4
            assert 1.1 * np.abs(s).max() < most and 1.1 * np.abs(p).max() < polynomial and polynomial >= abs(a)
            s = p * s


def test_log_probs_keep_their_operands_for_a_gradient_only():
    x, w, t, g = normal(1, 5, 4), normal(2, 4, 7), np.arange(5, dtype=np.int32), normal(3, 5)
    kept = lambda program, *args: [e.params['parts'] for e in mj.make_jaxpr(program)(*args).jaxpr.eqns if e.primitive.name == 'linear_log_probs']
    assert kept(lambda x, w: nn.linear_log_probs(x, w, t), x, w) == [False]
    assert kept(loss_program(False), x, w, t, g, g) == [True]

    def by_hand(x, w, t, g):
        outs = lax.linear_log_probs(x, w, t, with_parts=True)
        return lax.linear_log_probs_grad(x, w, t, outs[2], outs[3], g, parts=outs[4:]) + lax.linear_log_probs_grad(x, w, t, outs[2], outs[3], g)
    dx, dw, dx2, dw2 = evaluate(by_hand, x, w, t, g)
    assert np.array_equal(dx, dx2) and np.array_equal(dw, dw2)
    for rows in (5, 70):
        x, t, g = normal(1, rows, 4), np.arange(rows, dtype=np.int32) % 7, normal(3, rows)
        kept = [np.zeros(n, d) for n, d in K.linear_parts(x.shape, w.shape, False)]
        assert len(kept) == (1 if rows == 5 else 3)
        for at, v in enumerate(kept):
            for bad in (v[:-1], v.astype(np.uint32 if v.dtype == f32 else f32), v.reshape(1, -1)):
                refused(TypeError, lambda *a: lax.linear_log_probs_grad(*a[:5], parts=a[5:]), x, w, t, g, g, *(kept[:at] + [bad] + kept[at + 1:]))
        refused(TypeError, lambda *a: lax.linear_log_probs_grad(*a[:5], parts=a[5:]), x, w, t, g, g, *kept[:-1])
