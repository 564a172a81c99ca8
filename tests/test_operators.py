'''Group norm, log probabilities of tokens and linear recurrences, as programs: what is refused, what they and their gradients are
(the oracle against torch in 64 bits and against differences), and how they are planned.'''
import numpy as np
import pytest
import torch

from oracle import primitives as P
from oracle.eval_jaxpr import eval_closed_jaxpr
from vkjax_amd import minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

jnp, lax, nn = mj.numpy, mj.lax, mj.nn
f32 = np.float32
#a result that was computed in 64 bits and rounded once is off by at most half a step of fp32; what it was computed from in both
#places is the same, so twice that (and what 64 bits lose, which is nothing next to it)
ROUNDED = dict(rtol=2 * np.finfo(f32).eps / 2, atol=1e-30)


def evaluate(f, *args):
    return eval_closed_jaxpr(mj.make_jaxpr(f)(*args), *mj.tree_leaves(args))


def normal(seed, *shape, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(f32)


# ------------------------------------------------------------------ group norm

@pytest.mark.parametrize('activation', [None, 'relu', 'silu'])
@pytest.mark.parametrize('shape,groups', [((3, 5, 4, 6), 3), ((2, 8), 2), ((4, 7, 5), 5), ((1, 2, 2, 2, 4), 1)])
def test_group_norm_oracle_is_torchs(shape, groups, activation):
    c = shape[-1]
    x, scale, shift, g = normal(1, *shape), normal(2, c), normal(3, c), normal(4, *shape)
    t = [torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in (x, scale, shift)]
    moved = t[0].movedim(-1, 1)
    moved = moved if moved.dim() > 2 else moved[..., None]
    z = torch.nn.functional.group_norm(moved, groups, t[1], t[2], 1e-5)
    z = z.movedim(1, -1).reshape(shape)
    y = {None: lambda v: v, 'relu': torch.relu, 'silu': torch.nn.functional.silu}[activation](z)
    y.backward(torch.tensor(g, dtype=torch.float64))
    got = P.group_norm(x, scale, shift, groups, 1e-5, activation)
    assert np.allclose(got[0], y.detach().numpy(), rtol=1e-6, atol=1e-7)
    grads = P.group_norm_grad(g, x, scale, shift, got[1], got[2], groups, 1e-5, activation)
    for a, b in zip(grads, t):
        assert np.allclose(a, b.grad.numpy(), rtol=1e-6, atol=1e-6)


def test_group_norm_gradient_is_that_of_differences():
    x, scale, shift, g = normal(1, 2, 3, 3, 4), normal(2, 4), normal(3, 4), normal(4, 2, 3, 3, 4)

    def loss(x, scale, shift):
        _, z, _, _ = P._group_norm64(x, scale, shift, 2, 1e-5)
        return (P._activation64(z, 'silu')[0].reshape(g.shape) * g).sum()
    grads = P.group_norm_grad(g, x, scale, shift, None, None, 2, 1e-5, 'silu')
    for k, grad in enumerate(grads):
        for at in np.ndindex(*grad.shape):
            moved = [[v.astype(np.float64) for v in (x, scale, shift)] for _ in range(2)]
            moved[0][k][at] += 1e-5
            moved[1][k][at] -= 1e-5
            #a central difference is off by the third derivative times 1e-10, and 64 bits' rounding over 1e-5
            assert abs((loss(*moved[0]) - loss(*moved[1])) / 2e-5 - grad[at]) < 1e-5 * max(1, abs(grad[at]))


@pytest.mark.parametrize('change,error', [
    (dict(groups=5), ValueError), (dict(groups=0), ValueError), (dict(eps=0.0), ValueError), (dict(eps=np.inf), ValueError),
    (dict(activation='tanh'), ValueError), (dict(scale=np.ones(7, f32)), TypeError), (dict(shift=np.ones((1, 6), f32)), TypeError),
    (dict(x=np.ones(6, f32)), TypeError), (dict(x=np.ones((3, 6), np.int32)), TypeError), (dict(scale=np.ones(6, bool)), TypeError)])
def test_group_norm_refuses(change, error):
    given = dict(dict(x=np.ones((3, 4, 6), f32), scale=np.ones(6, f32), shift=np.ones(6, f32), groups=3, eps=1e-5, activation=None), **change)
    with pytest.raises(error):
        mj.make_jaxpr(lambda x, scale, shift: nn.group_norm(x, scale, shift, given['groups'], given['eps'], given['activation']))(
            given['x'], given['scale'], given['shift'])


# ------------------------------------------------------------------ log probabilities of tokens

def torch_log_probs(logits, tokens, top):
    '''64-bit results and the function that sums them up with cotangents, by torch.'''
    z = torch.tensor(logits, dtype=torch.float64, requires_grad=True)
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    entropy = -(p * logp.masked_fill(p == 0, 0.0)).sum(-1)
    token = torch.tensor(np.asarray(tokens, np.int64))
    best = torch.argsort(z.detach(), dim=-1, descending=True, stable=True)[..., :top]
    return z, logp.gather(-1, token[..., None])[..., 0], entropy, logp.gather(-1, best), best


@pytest.mark.parametrize('top', [0, 1, 5])
@pytest.mark.parametrize('shape', [(7, 11), (2, 3, 40), (9,)])
def test_log_probs_oracle_is_torchs(shape, top):
    logits = normal(1, *shape, scale=3.0)
    logits.reshape(-1)[::4] = np.round(logits.reshape(-1)[::4])                    #some equal scores
    tokens = np.random.default_rng(2).integers(0, shape[-1], shape[:-1]).astype(np.int32)
    z, lp, entropy, top_lp, best = torch_log_probs(logits, tokens, top)
    got = P.token_log_probs(logits, tokens, top)
    assert np.allclose(got[0], lp.detach(), **ROUNDED) and np.allclose(got[1], entropy.detach(), rtol=1e-6)
    g = [normal(k, *shape[:-1]) for k in (3, 4)] + ([normal(5, *shape[:-1], top)] if top else [])
    if top:
        assert np.allclose(got[3], top_lp.detach(), **ROUNDED) and np.array_equal(got[4], best)
    total = sum((torch.tensor(a, dtype=torch.float64) * b).sum() for a, b in zip(g, (lp, entropy, top_lp)))
    total.backward()
    cts = g[:2] + ([g[2], got[4]] if top else [])
    d = P.token_log_probs_grad(logits, tokens, got[2], got[1], *cts, has_log_probs=True, has_entropy=True, top=top)
    assert np.allclose(d, z.grad, rtol=1e-6, atol=1e-7)


def test_log_probs_gradient_is_that_of_differences():
    logits, tokens = normal(1, 3, 5), np.array([4, -1, 0], np.int32)
    g = [normal(2, 3), normal(3, 3), normal(4, 3, 2)]
    which = P.token_log_probs(logits, tokens, 2)[4]

    def loss(z):
        _, token, given, _, logp, p = P._token_rows64(z, tokens)
        rows = np.arange(3)
        value = g[0] * logp[rows, token] - g[1] * (p * logp).sum(1) + (g[2] * np.take_along_axis(logp, np.maximum(which, 0), 1)).sum(1)
        return (value * given).sum()
    d = P.token_log_probs_grad(logits, tokens, None, None, *g, which, has_log_probs=True, has_entropy=True, top=2)
    for at in np.ndindex(3, 5):
        up, down = logits.astype(np.float64), logits.astype(np.float64)
        up[at] += 1e-5
        down[at] -= 1e-5
        assert abs((loss(up) - loss(down)) / 2e-5 - d[at]) < 1e-5


def test_log_probs_of_masked_padded_and_broken_rows():
    inf, nan = np.inf, np.nan
    logits = np.array([[0, -inf, 0, 0], [-inf] * 4, [1, 2, nan, 4], [1, inf, 2, 3], [nan] * 4, [-inf, -inf, 5, -inf]], f32)
    lp, entropy, _, top_lp, top = P.token_log_probs(logits, np.array([1, 2, 0, 0, -100, 2], np.int32), 2)
    assert lp[0] == -inf and np.isclose(entropy[0], np.log(3)) and top[0].tolist() == [0, 2]
    assert lp[1] == -inf and entropy[1] == 0 and top[1].tolist() == [0, 1] and (top_lp[1] == -inf).all()
    assert np.isnan(lp[2]) and np.isnan(entropy[2]) and top[2].tolist() == [2, 3]
    assert np.isnan(lp[3]) and np.isnan(entropy[3]) and top[3].tolist() == [1, 3]
    assert lp[4] == 0 and entropy[4] == 0 and top[4].tolist() == [-1, -1] and (top_lp[4] == 0).all()
    assert lp[5] == 0 and entropy[5] == 0 and top[5].tolist() == [2, 0] and top_lp[5].tolist() == [0, -inf]


@pytest.mark.parametrize('logits,tokens,top,error', [
    (np.ones((3, 4), f32), np.zeros(3, np.int32), 5, ValueError), (np.ones((3, 40), f32), np.zeros(3, np.int32), 33, ValueError),
    (np.ones((3, 4), f32), np.zeros(3, np.int32), -1, ValueError), (np.ones((3, 4), f32), np.zeros(3, f32), 0, TypeError),
    (np.ones((3, 4), f32), np.zeros((3, 1), np.int32), 0, TypeError), (np.ones((3, 0), f32), np.zeros(3, np.int32), 0, TypeError),
    (np.ones((3, 4), np.int32), np.zeros(3, np.int32), 0, TypeError), (np.ones((), f32), np.zeros((), np.int32), 0, TypeError),
    (np.ones((3, 4), f32), np.zeros(3, bool), 0, TypeError)])
def test_log_probs_refuse(logits, tokens, top, error):
    with pytest.raises(error):
        mj.make_jaxpr(lambda z, t: nn.token_log_probs(z, t, top))(logits, tokens)


# ------------------------------------------------------------------ recurrences

def torch_recurrence(factor, x, state, lengths, reverse, gated):
    t = [torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in (factor, x, state)]
    now, hs = t[2], [None] * x.shape[1]
    order = range(x.shape[1])
    for k in (reversed(order) if reverse else order):
        a = torch.sigmoid(t[0][:, k]) if gated else t[0][:, k]
        new = a * now + ((1 - a) * t[1][:, k] if gated else t[1][:, k])
        inside = torch.tensor(k < np.asarray(lengths))[:, None]
        now = hs[k] = torch.where(inside, new, now)
    return t, torch.stack(hs, 1) if hs else t[1], now


@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('lengths', [[6, 6, 6], [6, 0, 3], [1, 99, -4]])
def test_recurrence_oracle_is_torchs(gated, reverse, lengths):
    factor, x, state = normal(1, 3, 6, 4), normal(2, 3, 6, 4), normal(3, 3, 4)
    lengths = np.array(lengths, np.int32)
    t, h, last = torch_recurrence(factor, x, state, lengths, reverse, gated)
    params = dict(gated=gated, reverse=reverse, has_state=True, has_lengths=True)
    got = P.linear_recurrence(factor, x, state, lengths, **params)
    assert np.allclose(got[0], h.detach(), **ROUNDED) and np.allclose(got[1], last.detach(), **ROUNDED)
    g, g_last = normal(4, 3, 6, 4), normal(5, 3, 4)
    ((h * torch.tensor(g)).sum() + (last * torch.tensor(g_last)).sum()).backward()
    grads = P.linear_recurrence_grad(got[0], factor, x, state, lengths, g, g_last, has_g=True, has_last=True, **params)
    for a, b in zip(grads, t):
        assert np.allclose(a, b.grad, rtol=1e-6, atol=1e-7)


def test_recurrence_gradient_is_that_of_differences():
    factor, x, state = normal(1, 2, 4, 2), normal(2, 2, 4, 2), normal(3, 2, 2)
    g, g_last = normal(4, 2, 4, 2), normal(5, 2, 2)

    def loss(factor, x, state):
        now, total = state, 0.0
        for k in range(4):
            a = 1 / (1 + np.exp(-factor[:, k]))
            now = a * now + (1 - a) * x[:, k]
            total += (now * g[:, k]).sum()
        return total + (now * g_last).sum()
    flags = dict(gated=True, reverse=False, has_state=True, has_lengths=False)
    h, _ = P.linear_recurrence(factor, x, state, **flags)
    grads = P.linear_recurrence_grad(h, factor, x, state, g, g_last, has_g=True, has_last=True, **flags)
    for k, grad in enumerate(grads):
        for at in np.ndindex(*grad.shape):
            moved = [[v.astype(np.float64) for v in (factor, x, state)] for _ in range(2)]
            moved[0][k][at] += 1e-5
            moved[1][k][at] -= 1e-5
            assert abs((loss(*moved[0]) - loss(*moved[1])) / 2e-5 - grad[at]) < 1e-5 * max(1, abs(grad[at]))


@pytest.mark.parametrize('change', [
    dict(factor=np.ones((2, 3, 5), f32)), dict(x=np.ones((2, 12), f32), factor=np.ones((2, 12), f32)), dict(state=np.ones((2, 3), f32)),
    dict(state=np.ones((2, 4), np.int32)), dict(lengths=np.ones(3, np.int32)), dict(lengths=np.ones(2, np.uint32)),
    dict(lengths=np.ones(2, f32)), dict(lengths=np.ones((2, 1), np.int32)), dict(x=np.ones((2, 3, 4), np.int32)), dict(factor=np.ones((2, 3, 4), bool))])
def test_recurrences_refuse(change):
    given = dict(dict(factor=np.ones((2, 3, 4), f32), x=np.ones((2, 3, 4), f32), state=np.ones((2, 4), f32), lengths=np.ones(2, np.int32)), **change)
    for f in (nn.gated_recurrence, lax.linear_recurrence):
        with pytest.raises(TypeError):
            mj.make_jaxpr(lambda a, b, s, n: f(a, b, s, n))(given['factor'], given['x'], given['state'], given['lengths'])


# ------------------------------------------------------------------ differentiation

def test_vjp_is_the_gradient_of_the_weighted_sum():
    x, w, g = normal(1, 4, 3), normal(2, 3, 5), normal(3, 4, 5)

    def by_vjp(x, w, g):
        y, pullback = mj.vjp(lambda a, b: jnp.tanh(jnp.dot(a, b)), x, w)
        return (y,) + pullback(g)

    def by_grad(x, w, g):
        return (jnp.tanh(jnp.dot(x, w)),) + mj.grad(lambda a, b, c: jnp.sum(jnp.tanh(jnp.dot(a, b)) * c), argnums=(0, 1))(x, w, g)
    for a, b in zip(evaluate(by_vjp, x, w, g), evaluate(by_grad, x, w, g)):
        assert np.allclose(a, b, rtol=1e-6, atol=1e-7)


def test_vjp_of_one_value_in_two_places_and_of_several_results():
    x, g = normal(1, 4), normal(2, 4)

    def f(x, g):
        (y, z), pullback, aux = mj.vjp(lambda a, b: ((a * b, a + a), a * 2.0), x, x, has_aux=True)
        return (aux,) + pullback((g, g))
    aux, da, db = evaluate(f, x, g)
    assert np.allclose(aux, 2 * x) and np.allclose(da, g * x + 2 * g) and np.allclose(db, g * x)


def test_vjp_of_an_unused_argument_and_a_plain_cotangent():
    def f(x, y):
        out, pullback = mj.vjp(lambda a, b: {'s': a * 3.0}, x, y)
        return pullback({'s': np.ones(4, f32)})
    da, db = evaluate(f, normal(1, 4), normal(2, 2))
    assert (da == 3).all() and (db == 0).all() and db.shape == (2,)


def test_values_of_an_enclosing_function_are_constants():
    x, w = normal(1, 4), normal(2, 4)

    def f(x, w):
        inner = mj.jit(lambda a: a * w + x)                               #two levels down
        (y, pullback), d = mj.vjp(lambda a: inner(a) * x, x), mj.grad(lambda a: jnp.sum(a * x * w))(x)
        out, same = mj.vjp(lambda a: (w, a), x)
        return y, pullback(x)[0], d, out[0], same((w, x))[0]
    y, dx, d, out, same = evaluate(f, x, w)
    assert np.allclose(y, (x * w + x) * x) and np.allclose(dx, w * x * x) and np.allclose(d, x * w) and np.array_equal(out, w) and np.array_equal(same, x)
    JaxprInterpreter(mj.make_jaxpr(f)(x, w), plan_only=True)
    with pytest.raises(NotImplementedError):
        mj.make_jaxpr(lambda a: mj.make_jaxpr(lambda b: b + a)(np.ones(4, f32)))(x)
    kept = []
    mj.make_jaxpr(lambda a: kept.append(a) or a)(x)
    with pytest.raises(NotImplementedError):
        mj.make_jaxpr(lambda a: a + kept[0])(x)


@pytest.mark.parametrize('cotangent', [np.ones(3, f32), np.ones(4, np.int32), (np.ones(4, f32),)])
def test_vjp_refuses_cotangents_that_do_not_belong(cotangent):
    with pytest.raises(TypeError):
        mj.make_jaxpr(lambda x: mj.vjp(lambda a: a * 2.0, x)[1](cotangent))(np.ones(4, f32))


def test_vjp_refuses_results_that_are_no_floats():
    with pytest.raises(TypeError):
        mj.make_jaxpr(lambda x: mj.vjp(lambda a: jnp.argmax(a), x)[0])(np.ones(4, f32))


@pytest.mark.parametrize('with_top', [False, True])
def test_gradients_of_some_of_the_results(with_top):
    '''Results that the loss does not use have no cotangent.'''
    logits, tokens = normal(1, 4, 7), np.array([1, 2, -1, 6], np.int32)

    def loss(z, t):
        lp, entropy, top_lp, _ = nn.token_log_probs(z, t, 2)
        return jnp.sum(top_lp * 0.5) if with_top else -jnp.mean(lp)
    (d,) = evaluate(mj.grad(loss), logits, tokens)
    z, lp, _, top_lp, _ = torch_log_probs(logits, np.maximum(tokens, 0), 2)
    given = torch.tensor(tokens >= 0)
    ((top_lp * 0.5 * given[:, None]).sum() if with_top else -(lp * given).mean()).backward()
    assert np.allclose(d, z.grad, rtol=1e-6, atol=1e-7)

    def last_only(a, x):
        return jnp.sum(nn.gated_recurrence(a, x)[1])
    gate, x = normal(2, 2, 5, 3), normal(3, 2, 5, 3)
    da, dx = evaluate(mj.grad(last_only, argnums=(0, 1)), gate, x)
    t, _, last = torch_recurrence(gate, x, np.zeros((2, 3), f32), [5, 5], False, True)
    last.sum().backward()
    assert np.allclose(da, t[0].grad, rtol=1e-6, atol=1e-7) and np.allclose(dx, t[1].grad, rtol=1e-6, atol=1e-7)


# ------------------------------------------------------------------ plans

def token_model(params, tokens, targets, lengths):
    '''Embedding, gated recurrence, group norm per position, scores: the mean log probability of the targets.'''
    b, t = tokens.shape
    x = params['table'][tokens]
    c = x.shape[-1]
    flat = jnp.reshape(x, (b * t, c))
    gate = jnp.reshape(jnp.dot(flat, params['wg']) + params['bg'], (b, t, c))
    h, last = nn.gated_recurrence(gate, x, params['state'], lengths)
    y = nn.group_norm(jnp.reshape(h, (b * t, c)), params['scale'], params['shift'], 4, activation='silu')
    lp, entropy = nn.token_log_probs(jnp.reshape(jnp.dot(y, params['wo']), (b, t, params['wo'].shape[1])), targets)
    return -jnp.mean(lp) - 0.01 * jnp.mean(entropy), last


def token_model_inputs(b=3, t=9, c=16, v=50, seed=0):
    rng = np.random.default_rng(seed)
    params = dict(table=normal(seed, v, c), wg=normal(seed + 1, c, c, scale=0.3), bg=np.ones(c, f32), state=normal(seed + 2, b, c),
                  scale=0.5 + rng.random(c, dtype=f32), shift=normal(seed + 3, c, scale=0.1), wo=normal(seed + 4, c, v, scale=0.3))
    tokens = rng.integers(0, v, (b, t)).astype(np.int32)
    lengths = np.array([t - 2 * i for i in range(b)], np.int32)
    targets = np.where(np.arange(t) < lengths[:, None], rng.integers(0, v, (b, t)), -1).astype(np.int32)
    return params, tokens, targets, lengths


def token_model_step(params, tokens, targets, lengths):
    (loss, last), grads = mj.value_and_grad(token_model, has_aux=True)(params, tokens, targets, lengths)
    return loss, last, grads


@pytest.mark.parametrize('fuse', [True, False])
@pytest.mark.parametrize('two_lanes', [True, False])
def test_a_token_model_is_planned(fuse, two_lanes):
    program = JaxprInterpreter(mj.make_jaxpr(token_model_step)(*token_model_inputs()), plan_only=True, fuse=fuse, two_lanes=two_lanes)
    for op, launch in zip(program.all_ops, program.launches):
        assert all(g >= 1 for g in launch.grid) and launch.grid[1] <= 65535 and launch.grid[0] * launch.block[0] < 2**32
        for i, (b, _) in enumerate(launch.buffers):
            assert b is None or b.tensor is not None, (launch.kernel, i)
        if op.meta is not None and op.meta[0] == 'operator':
            #nothing a launch writes stands where something it reads stands
            written = {id(launch.buffers[i][0].tensor) for i in launch.written if launch.buffers[i][0] is not None}
            read = {id(b.tensor) for i, (b, _) in enumerate(launch.buffers) if b is not None and i not in launch.written}
            assert not written & read, launch.kernel


def test_unused_operators_are_not_launched():
    def f(x, scale, shift, logits, tokens):
        nn.group_norm(x, scale, shift, 2)
        nn.gated_recurrence(x, x)
        nn.token_log_probs(logits, tokens, 3)
        return scale * 2.0
    program = JaxprInterpreter(mj.make_jaxpr(f)(normal(1, 2, 5, 4), normal(2, 4), normal(3, 4), normal(4, 3, 9), np.zeros(3, np.int32)), plan_only=True)
    assert [l.kernel.startswith('ew') or 'affine' in l.kernel for l in program.launches] == [True], [l.kernel for l in program.launches]


def test_arrays_without_elements_are_planned():
    def norm(x, scale, shift, g):
        y, pullback = mj.vjp(lambda *a: nn.group_norm(*a, 2), x, scale, shift)
        return (y,) + pullback(g)
    for shape in ((0, 5, 4), (3, 0, 4)):
        x = np.zeros(shape, f32)
        y, dx, dscale, dshift = evaluate(norm, x, np.ones(4, f32), np.ones(4, f32), x)
        assert y.shape == dx.shape == shape and not dscale.any() and not dshift.any()
        JaxprInterpreter(mj.make_jaxpr(norm)(x, np.ones(4, f32), np.ones(4, f32), x), plan_only=True)

    def recurrence(gate, x, state, g, g_last):
        outs, pullback = mj.vjp(nn.gated_recurrence, gate, x, state)
        return tuple(outs) + pullback((g, g_last))
    for shape in ((0, 5, 4), (3, 0, 4), (3, 5, 0)):
        x, state, g_last = np.zeros(shape, f32), normal(1, shape[0], shape[2]), normal(2, shape[0], shape[2])
        h, last, dgate, dx, dstate = evaluate(recurrence, x, x, state, x, g_last)
        assert np.array_equal(last, state) and np.array_equal(dstate, g_last) and dgate.shape == shape
        JaxprInterpreter(mj.make_jaxpr(recurrence)(x, x, state, x, g_last), plan_only=True)

    def probs(z, t, g):
        outs, pullback = mj.vjp(lambda v: nn.token_log_probs(v, t), z)
        return tuple(outs) + pullback((g, g))
    z, t = np.zeros((0, 7), f32), np.zeros(0, np.int32)
    assert evaluate(probs, z, t, np.zeros(0, f32))[2].shape == (0, 7)
    JaxprInterpreter(mj.make_jaxpr(probs)(z, t, np.zeros(0, f32)), plan_only=True)


# ------------------------------------------------------------------ gradients called by themselves

def refused(error, f, *args):
    with pytest.raises(error):
        mj.make_jaxpr(f)(*args)


@pytest.mark.parametrize('which,shape', [(0, (2, 5, 12)), (1, (2, 6, 8)), (2, (8,)), (3, (11,)), (3, (12, 1)), (4, (2, 4)), (4, (3, 3)), (5, (2,))])
def test_group_norm_gradient_refuses_shapes_that_do_not_belong(which, shape):
    shapes = [(2, 6, 12), (2, 6, 12), (12,), (12,), (2, 3), (2, 3)]
    mj.make_jaxpr(lambda *a: lax.group_norm_grad(*a, 3))(*[np.zeros(s, f32) for s in shapes])
    shapes[which] = shape
    refused((TypeError, ValueError), lambda *a: lax.group_norm_grad(*a, 3), *[np.zeros(s, f32) for s in shapes])


def test_group_norm_gradient_refuses_what_group_norm_refuses():
    arrays = [np.zeros(s, f32) for s in [(2, 6, 12), (2, 6, 12), (12,), (12,), (2, 5), (2, 5)]]
    refused(ValueError, lambda *a: lax.group_norm_grad(*a, 5), *arrays)
    arrays[4:] = [np.zeros((2, 3), f32)] * 2
    refused(ValueError, lambda *a: lax.group_norm_grad(*a, 3, eps=1e-60), *arrays)
    refused(ValueError, lambda *a: lax.group_norm(*a, 3, eps=1e-60), *arrays[1:4])
    refused(ValueError, lambda *a: lax.group_norm_grad(*a, 3, activation='tanh'), *arrays)
    for k in range(6):
        refused(TypeError, lambda *a: lax.group_norm_grad(*a, 3), *[v.astype(np.int32) if i == k else v for i, v in enumerate(arrays)])


def test_log_probs_gradient_refuses():
    z, t, row, top, ids = np.zeros((3, 9), f32), np.zeros(3, np.int32), np.zeros(3, f32), np.zeros((3, 2), f32), np.zeros((3, 2), np.int32)
    mj.make_jaxpr(lax.token_log_probs_grad)(z, t, row, row, row, row, top, ids)
    for args in [(z, t[:2], row, row, row), (z, t, row[:2], row, row), (z, t, row, row, row[:1]), (z, t, row, row, row, row, top, ids[:, :1]), (z, row, row, row, row),
                 (z, t, row, row, t), (z, t, t, row, row), (z, t, row, row, row, row, ids, ids), (z, t, row, row, row, row, top, top), (z.astype(np.int32), t, row, row, row),
                 (z, t, row, row, row, row, top[:, :0], ids[:, :0]), (z[:, :0], t, row, row, row)]:
        refused(TypeError, lax.token_log_probs_grad, *args)


def test_recurrence_gradient_refuses():
    x, last = np.zeros((2, 5, 3), f32), np.zeros((2, 3), f32)
    mj.make_jaxpr(lambda *a: lax.linear_recurrence_grad(*a[:4], None, *a[4:]))(x, x, x, last, x, last)
    for k, bad in [(0, x[:, :4]), (0, x.astype(np.int32)), (1, x[:1]), (2, x[..., :2]), (3, last[:1]), (4, x[:, 1:]), (4, x.astype(np.int32)), (5, last[:, :1]), (5, x)]:
        args = [x, x, x, last, x, last]
        args[k] = bad
        refused(TypeError, lambda *a: lax.linear_recurrence_grad(*a[:4], None, *a[4:]), *args)
    refused(TypeError, lambda f, x: lax.linear_recurrence_grad(None, f, x), x, x)


def test_gradients_have_no_gradients_of_their_own():
    x, s = np.zeros((2, 6, 12), f32), np.ones(12, f32)

    def twice(x, s):
        inner = lambda x: lax.add(mj.numpy.sum(mj.grad(lambda v: mj.numpy.sum(nn.group_norm(v, s, s, 3)))(x)), np.float32(0))
        return mj.grad(inner)(x)
    refused(NotImplementedError, twice, x, s)


def test_gradients_through_nested_jits():
    x, s, b = normal(1, 2, 6, 12), normal(2, 12), normal(3, 12)

    def norm(*a):
        return nn.group_norm(*a, 3, activation='silu')

    def with_gradient(f):
        def g(*a):
            y, pullback = mj.vjp(f, *a)
            return (y,) + pullback(y)
        return g
    run = lambda f: eval_closed_jaxpr(mj.make_jaxpr(f)(x, s, b), x, s, b)
    plain = run(with_gradient(norm))
    for other in (with_gradient(mj.jit(norm)), lambda *a: mj.jit(with_gradient(norm))(*a), lambda *a: mj.jit(with_gradient(lambda *q: mj.jit(norm)(*q)))(*a)):
        assert all(np.array_equal(p, q) for p, q in zip(run(other), plain))
        JaxprInterpreter(mj.make_jaxpr(other)(x, s, b), plan_only=True)
