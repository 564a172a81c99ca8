'''Gradients through functions with derivative rules of their own, and of values that a program passes in several places: which operand a
cotangent belongs to.'''
import numpy as np
import pytest

from oracle.eval_jaxpr import eval_closed_jaxpr
from vkjax_amd import minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

jnp, lax, nn = mj.numpy, mj.lax, mj.nn
f32 = np.float32
X, W = np.array([1, 2, 3], f32), np.array([4, 5, 6], f32)


def evaluate(f, *args):
    closed = mj.make_jaxpr(f)(*args)
    JaxprInterpreter(closed, plan_only=True)
    return eval_closed_jaxpr(closed, *mj.tree_leaves(args))


def with_rule(f, rule):
    h = mj.custom_jvp(f)
    h.defvjp(rule)
    return h


# ------------------------------------------------------------------ rules of functions that close over values

RULES = {'any': lambda g, y, *a: [g * f32(7)], 'fixed': lambda g, y, a: [g * f32(7)], 'default': lambda g, y, a, slope=f32(7): [g * slope]}


@pytest.mark.parametrize('rule', RULES.values(), ids=RULES)
@pytest.mark.parametrize('closed_over', ['traced', 'array', 'both', 'nested'])
def test_a_rule_gets_the_arguments_and_not_what_the_function_closes_over(rule, closed_over):
    def f(x, w):
        inner = {'traced': lambda a: a * w, 'array': lambda a: a * W, 'both': lambda a: a * w + W,
                 'nested': lambda a: mj.jit(lambda b: b * w)(a) - W}[closed_over]
        h = with_rule(inner, rule)
        y, pullback = mj.vjp(h, x)
        return mj.grad(lambda a: jnp.sum(h(a)))(x), mj.grad(lambda a: jnp.sum(mj.jit(h)(a) * a))(x), y, pullback(w)[0]
    d, product, y, pulled = evaluate(f, X, W)
    value = {'both': X * W + W, 'nested': X * W - W}.get(closed_over, X * W)
    assert np.array_equal(d, 7 * np.ones(3)) and np.array_equal(product, 7 * X + value) and np.array_equal(y, value) and np.array_equal(pulled, 7 * W)


def test_a_rule_of_two_arguments_and_a_value_that_is_closed_over():
    def f(x, w):
        h = with_rule(lambda a, b: a * b * w, lambda g, y, a, b: [g * b, g * a * f32(3)])
        return mj.grad(lambda a, b: jnp.sum(h(a, b)), argnums=(0, 1))(x, w)
    da, db = evaluate(f, X, W)
    assert np.array_equal(da, W) and np.array_equal(db, 3 * X)


def test_what_a_function_with_a_rule_closes_over_has_no_gradient_of_it():
    '''The rule says nothing about w: a gradient with respect to it is refused, not zero.'''
    def f(x, w):
        return mj.grad(lambda q: jnp.sum(with_rule(lambda a: a * q, lambda g, y, a: [g])(x)))(w)
    with pytest.raises(NotImplementedError, match='closes over'):
        mj.make_jaxpr(f)(X, W)
    #without a rule the function is differentiated like any other
    d, = evaluate(lambda x, w: mj.grad(lambda q: jnp.sum(mj.custom_jvp(lambda a: a * q)(x)))(w), X, W)
    assert np.array_equal(d, X)


# ------------------------------------------------------------------ one value in several places

def test_gradients_of_one_value_in_two_places():
    '''f(a, b) = a^2 b^3 at a = b = x: 2 x^4 and 3 x^4.'''
    f = lambda a, b: jnp.sum(a * a * b * b * b)
    first, = evaluate(lambda x: mj.grad(f)(x, x), X)
    second, = evaluate(lambda x: mj.grad(f, argnums=1)(x, x), X)
    both = evaluate(lambda x: mj.grad(f, argnums=(0, 1))(x, x), X)
    value, *of_leaves = evaluate(lambda x: mj.value_and_grad(lambda p: f(*p))([x, x]), X)
    assert np.array_equal(first, 2 * X ** 4) and np.array_equal(second, 3 * X ** 4) and value == (X ** 5).sum()
    for a, b in (both, of_leaves):
        assert np.array_equal(a, first) and np.array_equal(b, second)


@pytest.mark.parametrize('make', [lambda: np.array([1, 2, 3], f32), lambda: f32(3), lambda: 3.0], ids=['array', 'scalar', 'python'])
def test_gradients_of_one_constant_in_two_places(make):
    c = make()

    def f(y):
        return mj.grad(lambda a, b: jnp.sum(a * a * b * y), argnums=(0, 1))(c, c) + (mj.vjp(lambda a, b: jnp.sum(a * a * b * y), c, c)[1](f32(1)),)
    da, db, (va, vb) = mj.tree_unflatten(mj.tree_structure((0, 0, (0, 0))), evaluate(f, X))
    total = (lambda v: v) if np.ndim(c) else np.sum
    assert np.array_equal(da, total(2 * c * c * X)) and np.array_equal(db, total(c * c * X)) and np.array_equal(va, da) and np.array_equal(vb, db)


def test_a_constant_that_is_an_argument_and_closed_over():
    c = X.copy()
    d, pulled = evaluate(lambda y: (mj.grad(lambda a: jnp.sum(a * c * y))(c), mj.vjp(lambda a: a * c * y, c)[1](y)[0]), W)
    assert np.array_equal(d, c * W) and np.array_equal(pulled, c * W * W)


def test_a_recurrence_over_one_array_as_gate_and_as_input():
    x, g = np.random.default_rng(0).standard_normal((2, 5, 3)).astype(f32), np.random.default_rng(1).standard_normal((2, 5, 3)).astype(f32)
    f = lambda gate, x, g: mj.grad(lambda p, q: jnp.sum(nn.gated_recurrence(p, q)[0] * g), argnums=(0, 1))(gate, x)
    apart, together = evaluate(f, x, x, g), evaluate(lambda x, g: f(x, x, g), x, g)
    assert all(np.array_equal(a, b) for a, b in zip(apart, together)) and not np.array_equal(*apart)
    through_vjp = evaluate(lambda x, g: mj.vjp(lambda p, q: nn.gated_recurrence(p, q)[0], x, x)[1](g), x, g)
    assert all(np.array_equal(a, b) for a, b in zip(apart, through_vjp))


# ------------------------------------------------------------------ functions that hand an argument on

@pytest.mark.parametrize('f', [lambda a: a, lambda a: mj.jit(lambda b: b)(a)], ids=['itself', 'through a call'])
def test_a_rule_of_a_function_that_returns_its_argument(f):
    '''A gradient that is turned round or scaled on its way back: the function is the identity.'''
    h = with_rule(f, lambda g, y, a: [g * f32(-3)])
    d, twice, beside, constant = evaluate(lambda x: (mj.grad(lambda a: jnp.sum(h(a)))(x), mj.grad(lambda a: jnp.sum(h(h(a)) * a))(x),
                                                     mj.grad(lambda a: jnp.sum(h(a) + a))(x), mj.grad(lambda a: jnp.sum(h(a)))(W)), X)
    assert (d == -3).all() and np.array_equal(twice, 9 * X + X) and (beside == -2).all() and (constant == -3).all()


# ------------------------------------------------------------------ the log of the sum, and the rest of it

def test_gradients_of_log_probabilities_have_the_log_of_the_sum_unrounded():
    rng = np.random.default_rng(0)
    z, t, g = (rng.standard_normal((5, 9)) * 2 + 1e4).astype(f32), np.array([0, 8, -1, 3, 9], np.int32), rng.standard_normal(5).astype(f32)
    z[3] = -np.inf

    def f(z, t, g):
        inside = mj.jit(lambda v: nn.token_log_probs(v, t)[0])
        return mj.vjp(inside, z)[1](g), mj.vjp(lambda v: nn.token_log_probs(v, t, 2)[2], z)[1](jnp.broadcast_to(jnp.reshape(g, (5, 1)), (5, 2)))

    closed = mj.make_jaxpr(f)(z, t, g)
    made  = [e.outvars[-1] for e in closed.jaxpr.eqns if e.primitive.name == 'token_log_probs']
    grads = [e for e in closed.jaxpr.eqns if e.primitive.name == 'token_log_probs_grad']
    assert len(made) == len(grads) == 2 and all(e.params['has_rest'] and e.invars[4] is rest for e, rest in zip(grads, made))
    lp, entropy, log_sum, top_lp, top, rest = evaluate(lambda z, t: lax.token_log_probs(z, t, 2, with_rest=True), z, t)
    assert all(np.array_equal(a, b) for a, b in zip((lp, entropy, log_sum, top_lp, top), evaluate(lambda z, t: lax.token_log_probs(z, t, 2), z, t)))
    z64 = z[[0, 1]].astype(np.float64)
    exact = z64.max(1) + np.log(np.exp(z64 - z64.max(1, keepdims=True)).sum(1))
    assert not rest[2:].any() and np.allclose(log_sum[:2].astype(np.float64) + rest[:2], exact, rtol=0, atol=1e-10) and rest[:2].all()
    #by itself, with the rest and without it
    alone = evaluate(lambda *a: lax.token_log_probs_grad(*a[:5], log_sum_rest=a[5]), z, t, log_sum, entropy, g, rest)[0]
    assert np.array_equal(alone, evaluate(lax.token_log_probs_grad, z, t, log_sum, entropy, g)[0])


def test_the_rest_of_the_log_of_the_sum_is_one_value_per_row():
    z, t, row = np.zeros((3, 9), f32), np.zeros(3, np.int32), np.zeros(3, f32)
    for bad in (row[:2], t, np.zeros((3, 1), f32)):
        with pytest.raises(TypeError):
            mj.make_jaxpr(lambda *a: lax.token_log_probs_grad(*a[:5], log_sum_rest=a[5]))(z, t, row, row, row, bad)
    with pytest.raises(NotImplementedError):
        mj.make_jaxpr(lambda z: mj.grad(lambda v: jnp.sum(lax.token_log_probs(v, t, 0, with_rest=True)[3]))(z))(z)
