'''How launches of short causal convolutions, selective scans, log probabilities from weights and orthogonalised matrices are cut: over the sizes of the tests on the GPU and over ranges of others
(nothing is allocated).'''
import os
import random

import numpy as np
import pytest

from tests.test_gpu_token_model_operators import CONVS, LOSSES, MATRICES, SCANS
from tests.test_operator_plans import TOOLS, buffer, kernels_of, log_int, scratch
from vkjax_amd import kernels as K, minijax as mj
from vkjax_amd.csrc import build
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

MODULES = ('causal_conv', 'selective_scan', 'linear_log_probs', 'orthogonalize')
f32 = np.float32
nn = mj.nn


def zeroed(n, use):
    return buffer(n, dtype=np.uint32)


def conv_launches(b, t, c, k, gradient):
    x, w, row = buffer(b, t, c), buffer(k, c), buffer(c)
    if gradient:
        return K.causal_conv_grad(x, w, row, None, x, w, row, None, None, x, None, 'silu', scratch)
    return K.causal_conv(x, buffer(b, k - 1, c), x, w, row, None, None, None)


def scan_launches(b, t, c, n, gradient):
    x, a, m, row, state = buffer(b, t, c), buffer(c, n), buffer(b, t, n), buffer(c), buffer(b, c, n)
    kept = buffer(-(-t // K.SELECTIVE_SCAN_KEPT), b, n, c)
    if gradient:
        return K.selective_scan_grad(x, x, a, m, m, row, None, state, row, kept, x, x, a, m, m, row, None, None, row, x, state, True, scratch)
    return K.selective_scan(x, state, None, x, x, a, m, m, row, None, state, None, row, True, scratch)


def loss_launches(rows, h, v, transposed, gradient, keeping=True):
    x, w, t, r = buffer(rows, h), buffer(*((v, h) if transposed else (h, v))), buffer(rows, dtype=np.int32), buffer(rows)
    parts = [buffer(n, dtype=d) for n, d in K.linear_parts(x.shape, w.shape, transposed)] if keeping else None
    if gradient:
        return K.linear_log_probs_grad(x, w, x, w, t, r, r, r, r, transposed, scratch, zeroed, parts)
    return K.linear_log_probs(r, r, r, r, x, w, t, transposed, scratch, zeroed, parts)


def matrix_launches(*shape, steps=3):
    x = buffer(*shape)
    return K.orthogonalize(x, x, steps, (3.4445, -4.7750, 2.0315), 1e-7, scratch, zeroed)


def check(launches):
    '''What every launch has to keep to: a grid of fewer than 2^32 threads, a block of 1024 at most.'''
    for launch in launches:
        assert launch.grid[0] >= 1 and launch.block[0] <= 1024 and launch.grid[0] * launch.grid[1] * launch.block[0] < 2**32, launch.kernel
        yield launch.kernel


def launched(seed=1, draws=4000):
    rng, names = random.Random(seed), set()
    for k in range(draws):
        b, t, c = log_int(rng, 1, 100), log_int(rng, 1, 20000), log_int(rng, 1, 5000)
        for gradient in (False, True):
            names.update(check(conv_launches(b, t, c, rng.randint(2, 8), gradient)))
            names.update(check(scan_launches(b, t, c, log_int(rng, 1, 64), gradient)))
            if k < draws // 8:
                names.update(check(loss_launches(log_int(rng, 1, 20000), log_int(rng, 1, 5000), log_int(rng, 1, 150000), rng.random() < 0.5, gradient, rng.random() < 0.5)))
        if k < draws // 2:
            n = log_int(rng, 1, 30)
            names.update(check(matrix_launches(*([n] if n > 1 else []), log_int(rng, 1, 6000), log_int(rng, 1, 6000))))
    return names


@pytest.mark.skipif(not (TOOLS and all(os.path.exists(build.hsaco_path(m)) for m in MODULES)), reason='no code object, or no tool to look into it')
def test_kernels_exist_and_every_one_is_reached(tmp_path):
    found = {}
    for module in MODULES:
        found.update(kernels_of(module, tmp_path))
    names = launched()
    assert names <= set(found), names - set(found)
    assert set(found) == names, set(found) - names
    #(where a contraction is shared, what adds up slices of tiles of 128 costs a few registers too many; three scans have a wave more a SIMD by it)
    assert all(bytes_ <= (64 if '_shared' in k or k in ('selective_scan_grad_n4_m2', 'selective_scan_grad_n4_m8', 'selective_scan_n8_m8') else 0) for k, (_, bytes_) in found.items()), {k: v for k, v in found.items() if v[1]}


def test_sizes_of_the_tests_on_the_gpu_reach_every_kernel():
    names = set()
    for shape, k, _ in CONVS + [((2, t, c), k, None) for k in range(2, 9) for t in (1, 37) for c in (9, 12)]:
        names.update(n for g in (False, True) for n in check(conv_launches(*shape, k, g)))
    for b, t, c, n, *_ in SCANS:
        names.update(k for g in (False, True) for k in check(scan_launches(b, t, c, n, g)))
    for size in LOSSES:
        names.update(k for g in (False, True) for transposed in (False, True) for k in check(loss_launches(*size, transposed, g)))
    for shape in MATRICES:
        names.update(check(matrix_launches(*shape)))
    #(kernels of products, shared and not, have tests that choose the plan)
    products = {f'{name}{k[0]}{shared}' for name in ('linear_scores', 'linear_q', 'linear_product_a', 'linear_product_b', *(f'orthogonal_{n}' for n in ('square', 'polynomial', 'next', 'last')))
                for k in K.HALF_KERNELS for shared in ('', '_shared')}
    assert launched() - names <= products, launched() - names - products


@pytest.mark.parametrize('rows,columns,n', [(1, 1, 1), (127, 4000, 1), (512, 512, 12), (4096, 4096, 1), (33, 70000, 3), (1, 1000003, 1)])
def test_shares_of_a_product_cover_it(rows, columns, n):
    '''Every tile is one of the whole ones or has its contraction covered by slices.'''
    for launch in matrix_launches(n, rows, columns):
        if not launch.kernel.startswith('orthogonal_') or launch.kernel in ('orthogonal_squares', 'orthogonal_pack'):
            continue
        words = np.frombuffer(launch.params, np.uint32).astype(np.int64)
        kind, m, width, k, tiles_m, tiles_n, tiles = words[:7]
        whole, slices = words[13:15]
        side = 128 if '_128' in launch.kernel else 64
        assert tiles_m == -(-m // side) and tiles_n == -(-width // side)
        assert tiles == (tiles_m * (tiles_m + 1) // 2 if kind < 2 else tiles_m * tiles_n)
        all_tiles = tiles * n
        assert launch.grid[0] == (all_tiles if slices == 1 else whole + (all_tiles - whole) * slices) and ('_shared' in launch.kernel) == (slices > 1)


def test_the_largest_sizes_are_planned_and_larger_ones_refused():
    list(check(conv_launches(1, 2**29, 8, 4, True)))
    list(check(conv_launches(2**23 - 1, 4, 4, 4, False)))
    for size in ((1, 2**30, 1), (2**24, 4, 256), (1, 1, 2**30)):
        with pytest.raises(NotImplementedError):
            list(check(conv_launches(*size, 4, False)))
        with pytest.raises(NotImplementedError):
            list(check(conv_launches(*size, 4, True)))
    list(check(scan_launches(1, 2**29, 64, 16, False)))
    list(check(scan_launches(2**18, 1, 512, 15, False)))
    for size in ((1, 2**30, 1, 1), (2**22, 1, 2**10, 16), (2**26, 2, 64, 1)):
        with pytest.raises(NotImplementedError):
            list(check(scan_launches(*size, False)))
    with pytest.raises(NotImplementedError):
        list(check(scan_launches(1, 2**30, 1, 1, True)))
    list(check(loss_launches(2**20, 2000, 4096, False, True)))
    list(check(loss_launches(8, 4096, 2**25, True, True)))
    for size in ((2**27, 8, 1000), (100, 2**27, 8), (100, 8, 2**27), (2**20, 2048, 1000), (2**20, 8, 2**20)):
        for gradient in (False, True):
            with pytest.raises(NotImplementedError):
                list(check(loss_launches(*size, False, gradient)))
    list(check(matrix_launches(2**15, 2**15)))
    list(check(matrix_launches(1000, 2**20 - 1)))
    for shape in ((2, 2**20), (2**19, 2**19), (10000, 4096, 4096)):
        with pytest.raises(NotImplementedError):
            matrix_launches(*shape)


def test_what_a_gradient_of_log_probs_holds_at_a_time():
    '''The scores' cotangents stay below the bytes of a piece, or are a single tile's.'''
    for rows, h, v in ((4096, 1024, 32000), (20000, 64, 130001), (321, 500, 50001), (2**20, 64, 5000)):
        taken = []

        def noting(shape, dtype=f32):
            taken.append(int(np.prod(shape, dtype=np.int64)) * 4)
            return scratch(shape, dtype)
        x, w, t, r = buffer(rows, h), buffer(h, v), buffer(rows, dtype=np.int32), buffer(rows)
        parts = [buffer(n, dtype=d) for n, d in K.linear_parts(x.shape, w.shape, False)]
        K.linear_log_probs_grad(x, w, x, w, t, r, r, r, r, False, noting, zeroed, parts)
        blocks = -(-rows // 32) * 32
        #q both ways, the operands of the other products, slices of dx
        assert max(taken) <= max(K.LINEAR_PIECE, 4 * 128 * (blocks + 128), 4 * (h + 32) * (v + 32), 4 * (h + 32) * (blocks + 32), 4 * 64 * rows * h), (taken, rows, h, v)


@pytest.mark.parametrize('rows', [20, 300])
@pytest.mark.parametrize('transposed', [False, True])
def test_products_that_nobody_reads_are_left_out(rows, transposed):
    '''Of weights that are not trained, and of rows that no gradient goes on from.'''
    h, v = 200, 5000
    x, w, t, r = buffer(rows, h), buffer(*((v, h) if transposed else (h, v))), buffer(rows, dtype=np.int32), buffer(rows)
    parts = [buffer(n, dtype=d) for n, d in K.linear_parts(x.shape, w.shape, transposed)]
    flops = [sum(launch.flops for launch in K.linear_log_probs_grad(dx, dw, x, w, t, r, r, r, r, transposed, scratch, zeroed, parts)) for dx, dw in ((x, w), (x, None), (None, w))]
    assert all(f < 0.75 * flops[0] for f in flops[1:]), flops


@pytest.mark.parametrize('which', [(0,), (1,), (0, 1)], ids=str)
@pytest.mark.parametrize('rows', [20, 300])
def test_a_program_computes_the_gradients_that_it_returns(rows, which):
    x, w, t, g = np.zeros((rows, 200), f32), np.zeros((200, 5000), f32), np.zeros(rows, np.int32), np.ones(rows, f32)

    def f(x, w):
        given = [x, w]
        return mj.vjp(lambda *a: nn.linear_log_probs(*(a[which.index(i)] if i in which else given[i] for i in range(2)), t)[0], *(given[i] for i in which))[1](g)
    launched = {launch.kernel for launch in JaxprInterpreter(mj.make_jaxpr(f)(x, w), plan_only=True).launches if launch is not None}
    products = {n for n in launched if n.startswith(('linear_product', 'linear_rows_d')) and n != 'linear_rows_ds'}
    if rows == 20:
        assert {n[:14] for n in products} == {('linear_rows_dx', 'linear_rows_dw')[i] for i in which}
    else:
        jobs = [launch for launch in JaxprInterpreter(mj.make_jaxpr(f)(x, w), plan_only=True).launches if launch is not None and launch.kernel.startswith('linear_product')]
        assert len(jobs) == len(which)
