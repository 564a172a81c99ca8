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
        scales = words[7:10] if launch.kernel.startswith(('orthogonal_square_', 'orthogonal_poly', 'orthogonal_next', 'orthogonal_last')) else words[-3:-2] if launch.kernel == 'orthogonal_pack' else ()
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


@pytest.mark.parametrize('transposed', [False, True])
@pytest.mark.parametrize('rows,h,v', [(4096, 1024, 32000), (20000, 64, 130001), (2**20, 64, 5000), (2000, 300, 200000), (70000, 2000, 1100)])
def test_a_gradient_of_log_probs_holds_no_scores(rows, h, v, transposed):
    '''Array by array: a piece of the scores' cotangents, slices of dx, x as an operand, sums of shared contractions. All scores would be more than a piece.'''
    assert 4 * rows * v > K.LINEAR_PIECE
    x, w, t, r = buffer(rows, h), buffer(*((v, h) if transposed else (h, v))), buffer(rows, dtype=np.int32), buffer(rows)
    parts = [buffer(n, dtype=d) for n, d in K.linear_parts(x.shape, w.shape, transposed)]
    taken = []

    def noting(shape, dtype=np.float32):
        taken.append(scratch(shape, dtype))
        return taken[-1]
    dx, dw = buffer(*x.shape), buffer(*w.shape)
    launches = K.linear_log_probs_grad(dx, dw, x, w, t, r, r, r, r, transposed, noting, zeroed, parts)
    of = lambda name, at: {id(l.buffers[at][0]): l.buffers[at][0] for l in launches if l.kernel.startswith(name) and l.buffers[at][0] is not None}
    size = lambda b: 4 * b.size
    q, = of('linear_q', 0).values()
    blocks = -(-rows // 32) * 32
    tile = 4 * K.HALF_TILE * blocks
    assert size(q) <= max(K.LINEAR_PIECE, tile)
    sums = {k: b for k, b in of('linear_product', 0).items() if b is not dx and b is not dw}
    tiles_x = -(-rows // K.HALF_TILE) * -(-h // K.HALF_TILE)
    assert all(size(b) <= 2 * K.HALF_CUS // tiles_x * 4 * rows * h for b in sums.values()) and len(sums) <= 1
    operands = {**of('linear_pack', 0), **of('linear_pack', 1), **of('linear_pack', 2)}
    assert all(size(b) <= 4 * blocks * (-(-h // 32) * 32) for b in operands.values())
    #(sums of shared contractions: at most a round of the machine's tiles in 64 slices)
    shared = {**of('linear_product', 1), **of('linear_q', 1)}
    assert all(size(b) <= 64 * 2**20 for b in shared.values())
    named = {id(q), *sums, *operands, *shared}
    assert all(size(b) <= 2**20 + 12 * rows for b in taken if id(b) not in named)
    assert all(size(b) < 4 * rows * v for b in taken if id(b) not in {*sums, *operands})
