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
