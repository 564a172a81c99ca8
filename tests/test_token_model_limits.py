'''Token models' operators at the ends of what they take: what is planned there, and what is refused (nothing is allocated).'''
import numpy as np
import pytest

from tests.test_operator_plans import buffer, scratch
from tests.test_operators import normal, refused
from tests.test_token_model_plans import check, conv_launches, loss_launches, matrix_launches, zeroed
from vkjax_amd import kernels as K, minijax as mj

jnp, lax = mj.numpy, mj.lax


@pytest.mark.parametrize('steps,coefficients', [(32, (0.25, 0.0, 0.0)), (8, (0.0, 0.5, 0.0)), (2, (0.0, 0.0, 1e-20)), (2, (1e-30, 0.0, 0.0)), (3, (0.0, 0.0, 0.0)), (32, (3.4445, -4.7750, 2.0315))])
def test_scales_of_polynomials_are_powers_that_fp32_has(steps, coefficients):
    '''Polynomials under which singular values come to next to nothing: 2^scale and 2^-scale are factors on the device, of which it makes those from 2^-126 to 2^126.'''
    x, seen = buffer(100, 100), 0
    for launch in K.orthogonalize(x, x, steps, coefficients, 1e-7, scratch, zeroed):
        words = np.frombuffer(launch.params, np.int32)
        scales = words[7:10] if launch.kernel.startswith(('orthogonal_square_', 'orthogonal_poly', 'orthogonal_next', 'orthogonal_last')) else words[-1:] if launch.kernel == 'orthogonal_pack' else ()
        assert all(-126 <= s <= 126 for s in scales), (launch.kernel, scales)
        seen += len(scales)
    assert seen == 1 + 9 * steps


def test_gradients_of_convolutions_of_many_channels():
    '''Sums over time go through a launch of 16 threads a channel and tap.'''
    for t, c, k in ((4, 2**26, 4), (1, 2**26, 3), (1, 2**29 + 4, 8), (1, 2**28 // 9 + 1, 8)):
        list(check(conv_launches(1, t, c, k, False)))
        with pytest.raises(NotImplementedError):
            list(check(conv_launches(1, t, c, k, True)))
        #(without the kernel's and the bias' gradients there is no such launch)
        x, w = buffer(1, t, c), buffer(k, c)
        launch, = K.causal_conv_grad(x, None, None, None, x, w, None, None, None, x, None, None, scratch)
        list(check([launch]))
    for c, k in ((2**28 // 9 - 64, 8), (2**28 // 5 - 64, 4)):
        list(check(conv_launches(1, 1, c, k, True)))


def test_matrices_of_few_rows_by_the_million():
    '''A Gram matrix has a block of up to 1024 threads.'''
    for shape in ((12_000_000, 20, 20), (6_000_000, 48, 48), (11_184_811, 17, 17), (6_000_000, 40, 48)):
        for steps in (2, 5):
            with pytest.raises(NotImplementedError):
                list(check(matrix_launches(*shape, steps=steps)))
    for shape in ((11_184_810, 17, 17), (16_000_000, 16, 16), (5_592_405, 48, 48), (2_000_000, 64, 256)):
        assert 'orthogonal_small' in list(check(matrix_launches(*shape)))


def test_log_probs_of_many_rows_of_few_features():
    '''16 rows have a block of 1024 threads of the launch that joins their tiles.'''
    for rows, h, v in ((2**26 - 15, 8, 100), (2**27 - 1, 4, 50)):
        for gradient in (False, True):
            with pytest.raises(NotImplementedError):
                list(check(loss_launches(rows, h, v, False, gradient)))
    for gradient in (False, True):
        list(check(loss_launches(2**26 - 16, 8, 100, False, gradient)))


def test_log_probs_over_a_hundred_million_tokens():
    '''Tiles of 64 would be more than a launch can have blocks: those of 128 are taken.'''
    for rows, h, v in ((559, 54, 134200629), (832, 3, 132375801), (890, 8, 2**27 - 1)):
        for gradient in (False, True):
            assert any(name.endswith('_128') for name in check(loss_launches(rows, h, v, False, gradient)))


def test_scores_that_are_kept_for_a_gradient_have_none():
    '''Of few rows linear_log_probs keeps the scores, as float32: what a program makes of them has no part in its gradient, so that it is refused.'''
    x, w, t = normal(1, 3, 8), normal(2, 8, 10), np.zeros(3, np.int32)
    for at in range(2, 5):
        refused(NotImplementedError, lambda x: mj.grad(lambda x: jnp.sum(lax.linear_log_probs(x, w, t, with_parts=True)[at]))(x), x)
        refused(NotImplementedError, lambda x: mj.grad(lambda x: (lambda outs: jnp.sum(outs[0]) + jnp.sum(outs[at]))(lax.linear_log_probs(x, w, t, with_parts=True)))(x), x)
