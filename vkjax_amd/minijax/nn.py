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
