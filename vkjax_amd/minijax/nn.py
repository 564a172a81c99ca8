'''Neural-network helpers as they appear in traced programs (relu under a custom-jvp
call, softmax as max / sub / exp / sum / div), so that the device path sees the same
primitive sequences as with `jax.nn`.'''
import numpy as np

from . import lax, numpy as mnp
from .tracer import custom_jvp


@custom_jvp
def relu(x):
    return mnp.maximum(x, 0)


@relu.defvjp
def _relu_vjp(g, ans, x):
    #jax.nn.relu's own rule: the cotangent passes where x > 0 (no share at x == 0). The test is made on the
    #result (max(x, 0) > 0 exactly where x > 0), so the backward pass does not keep the pre-activation alive
    shape = tuple(g.shape)
    zeros = lax.broadcast_in_dim(np.float32(0), shape, ()) if shape else np.float32(0)
    return (lax.select(lax.gt(ans, zeros), g, zeros),)


def softmax(x, axis=-1):
    unnormalized = mnp.exp(x - lax.stop_gradient(mnp.max(x, axis, keepdims=True)))
    return unnormalized / mnp.sum(unnormalized, axis, keepdims=True)


def log_softmax(x, axis=-1):
    shifted = x - lax.stop_gradient(mnp.max(x, axis, keepdims=True))
    return shifted - mnp.log(mnp.sum(mnp.exp(shifted), axis, keepdims=True))


def batch_norm_inference(x, scale, shift, mean, var, eps=1e-5):
    '''Inference-mode batch norm over the trailing (channel) axis, written the way
    flax/haiku modules of the period lower it: the per-channel factor first, then three
    full-size broadcasting passes.'''
    inv = scale * lax.rsqrt(var + np.float32(eps))
    return (x - mean) * inv + shift


def group_norm(x, scale, shift, groups, eps=1e-5, activation=None):
    '''Group norm over channels-last activations x [N, ..., C], with the activation behind it (None, 'relu' or 'silu', which is
    z * sigmoid(z)): every sample is normalised over its positions and the channels of each of `groups` runs of C / groups
    neighbouring channels, then scaled and shifted per channel. groups=1 on [tokens, C] is layer norm. Differentiable with
    respect to x, scale and shift.'''
    return lax.group_norm(x, scale, shift, groups, eps, activation)[0]


def token_log_probs(logits, tokens, top=0):
    '''Log probabilities of given tokens (or classes) under softmax(logits): logits [..., V], tokens int32 [...]. Returns
    (log_probs [...], entropy [...]), the entropy being that of each row's whole distribution, and with top > 0 (up to 32) also
    (..., top_log_probs [..., top], top_tokens int32 [..., top]): the most likely tokens, equal scores by their number.

    * A row whose token lies outside the vocabulary (negative, say) is padding: its log probability and entropy are 0, its
      alternatives have log probability 0 and token -1, no gradient comes from it, and its logits are not looked at.
    * Logits of -inf are masked: they have no probability and add nothing to the entropy. In a row where every logit is -inf each
      log probability is -inf, the entropy is 0 and the gradient is 0.
    * NaN and +inf make their row's log probabilities and entropy NaN; among the alternatives NaN counts as the largest score.

    Differentiable with respect to the logits, through log_probs, entropy and top_log_probs.'''
    log_probs, entropy, _, *alternatives = lax.token_log_probs(logits, tokens, top)
    return (log_probs, entropy, *alternatives)


def gated_recurrence(gate, x, state=None, lengths=None, reverse=False):
    '''A recurrence with a gate per channel over x [batch, time, channels]: h[t] = a[t] h[t-1] + (1 - a[t]) x[t],
    a = sigmoid(gate). Returns (h, the state [batch, channels] behind the last step), so that a sequence can go on later: `state`
    is where it starts (zeros if None), and time may be 1, or 0. `lengths` int32 [batch]: a padded batch, in which a sequence's
    state stays what it is from its length on (in h too) and what gate and x hold there is not looked at; `reverse`: from the last
    time to the first. Differentiable with respect to gate, x and state. `lax.linear_recurrence` takes factors and addends, and says
    what becomes of values that many small factors leave next to nothing of, and of infinite ones.'''
    return lax.linear_recurrence(gate, x, state, lengths, reverse, gated=True)


def causal_conv(x, kernel, bias=None, state=None, lengths=None, activation=None):
    '''A short causal convolution along time over x [batch, time, channels], channel by channel, with the activation behind it (None or 'silu'):
    y[:, t] = activation(bias + sum_k kernel[k] * x[:, t - width + 1 + k]) for a kernel [width, channels], width 2 to 8. Returns (y, the last
    width - 1 inputs [batch, width - 1, channels]), so that a sequence can go on later, token by token: `state` is what stands in front of it
    (zeros if None). `lengths` int32 [batch]: a padded batch, in which y is 0 from a sequence's length on, x is not looked at there, and the last
    inputs are those in front of the length. Differentiable with respect to x, kernel, bias and state.'''
    return lax.causal_conv(x, kernel, bias, state, lengths, activation)


def selective_scan(x, delta, a, b, c, d=None, gate=None, state=None, lengths=None, delta_bias=None, softplus=False):
    '''A selective state space over x [batch, time, channels], with `states` (1 to 64) states h per channel:
    h[t] = exp(w a) h[t-1] + w x[t] b[t], y[t] = (sum over the states of c[t] h[t] + d x[t]) * silu(gate[t]), where w = delta[t], or
    softplus(delta[t] + delta_bias) (`softplus`); delta and gate are [batch, time, channels], a [channels, states], b and c [batch, time, states],
    d and delta_bias [channels]; d, gate and delta_bias may be None. Returns (y, the state [batch, channels, states] behind the last step), so that a
    sequence can go on later, token by token: `state` is where it starts (zeros if None), and time may be 1, or 0. `lengths` int32 [batch]: a
    padded batch, in which a sequence's state stays and y is 0 from its length on, and nothing else is looked at there. Differentiable with respect to
    every float32 operand. `lax.selective_scan` says what long products of factors come to.'''
    return lax.selective_scan(x, delta, a, b, c, d, gate, state, lengths, delta_bias, softplus)


def linear_log_probs(x, weights, tokens, transposed=False):
    '''Log probabilities of given tokens (or classes) under softmax(x @ weights), without keeping the scores: x [..., hidden], weights [hidden, vocabulary], or with `transposed` the
    rows of an embedding, [vocabulary, hidden]; tokens int32 [...]. Returns (log_probs [...], log_sums [...]), the latter being log(sum(exp(scores))) of each row. A cross entropy is
    -log_probs; the gradient works the scores out again, a piece of the vocabulary at a time. (Of up to 64 rows it takes the scores of the forward pass.) For a gradient the forward pass
    keeps, until that is done, the weights and x once more as the products take them, or the scores of up to 64 rows.

    * A row whose token lies outside the vocabulary (negative, say) is padding: its results are 0, no gradient comes from it, and its x is not looked at.
    * Up to 64 rows are computed by fp32 products. With more, numbers are held to 2^-22 of themselves or 2^-51 of the largest of their operand (x's given rows, the weights), and sums are rounded an
      eighth as often, as long as no score is off by more than 2^-24 by the latter: where the largest magnitudes of x and of the weights, times one another and the features, pass 2^26, or a number is not
      finite, fp32 products take their place (at a third to a half of the speed). So a row does not depend on what the others hold.
    * The scores' cotangents, g p, are held in the same way for more than 64 rows, to 2^-51 of the row's larger cotangent: what tokens with probabilities below 2^-28 get has fewer bits, below 2^-52 none; and of dweights a row's part
      (its cotangent times its x) to 2^-51 of the largest row's.
    * Infinities and NaN are those of fp32 arithmetic: a NaN in a row of x makes that row's results NaN, one in the weights those of every row; a token whose weights make its score -inf has probability 0.

    Differentiable with respect to x and weights, through both results.'''
    return lax.linear_log_probs(x, weights, tokens, transposed)[:2]


def orthogonalize(x, steps=5, coefficients=lax.ORTHOGONALIZE_COEFFICIENTS, eps=1e-7):
    '''Every matrix of x [..., rows, columns] with its singular values brought to about 1, as an optimiser does it with the momentum of a weight's gradients before the weight is updated:
    x / (|x| + eps), then `steps` (1 to 32) times the polynomial a s + b s^3 + c s^5 of the singular values, by products of matrices. With the default coefficients five steps bring singular values
    from 0.01 of the norm on to between 0.7 and 1.2; (1.5, -0.5, 0) approaches 1 itself, more slowly. Matrices of zeros stay zeros; NaN and infinities in a matrix spoil that one only; one of up
    to 64 rows or columns whose norm (with eps) is below 1e-36 or beyond 1e36 may lose bits.
    Coefficients with which singular values do not stay small are refused. Not differentiable.'''
    return lax.orthogonalize(x, steps, coefficients, eps)
