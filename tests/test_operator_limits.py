'''Launches of group norms, log probabilities and recurrences at the largest sizes that their kernels address, as they are planned (nothing is
allocated).'''
import os

import numpy as np
import pytest

from tests.test_gpu_operator_kernels import NORM_SIZES, RECURRENCE_SIZES
from tests.test_operator_plans import TOOLS, buffer, check_log_probs, check_recurrence, kernels_of, norm_launches
from vkjax_amd import kernels as K, minijax as mj
from vkjax_amd.csrc import build
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

lax, nn, f32 = mj.lax, mj.nn, np.float32


# ------------------------------------------------------------------ recurrences: what a tile's descriptor covers

@pytest.mark.parametrize('b,t,c', [(1, 1, 2**29 - 4), (1, 1, 2**29 - 1), (2, 1, 2**28 - 2), (1, 4, 2**27 - 3), (1, 4, 2**27 - 4), (3, 2, 2**28 - 4), (1, 16, 2**25 - 8), (1, 300, 2**21 - 4),
                                   (1, 2000, 2**21 - 5)])
@pytest.mark.parametrize('gradient', [False, True])
def test_a_recurrences_tile_ends_before_the_place_of_lanes_without_an_element(b, t, c, gradient):
    '''Lanes without an element load and store at offset 2^31 of their tile's descriptor, which has to be behind its end.'''
    x, state = buffer(b, t, c), buffer(b, c)
    zeroed = lambda n, use: buffer(n, dtype=np.uint32)
    try:
        if gradient:
            launch, = K.linear_recurrence_grad(x, x, state, x, x, x, state, None, x, state, True, False, zeroed)
        else:
            launch, = K.linear_recurrence(x, state, x, x, state, None, True, False, zeroed)
    except NotImplementedError:
        return
    _, T, C, cstrips, strips, tiles, lines, of_each, log2_w, _ = np.frombuffer(launch.params, np.uint32).astype(np.int64)
    vec, steps = 4 if '_v4' in launch.kernel else 1, int(launch.kernel.split('_l')[1].split('_')[0])
    assert ((256 >> log2_w) * steps * C + (vec << log2_w)) * 4 < 2**31


def test_recurrences_below_that_are_planned():
    for b, t, c in ((1, 1, 2**28), (1, 4, 2**26), (1, 300, 2**18)):
        assert list(check_recurrence(b, t, c))


# ------------------------------------------------------------------ group norm of single positions: where pairs lie in shared memory

@pytest.mark.parametrize('n,groups,cg', [(1, 1, 3), (1, 1, 5), (5, 1, 255), (3000, 1, 255), (7, 3, 85), (1, 5, 51), (2, 1, 4), (8191, 16, 65)])
def test_statistics_of_rows_lie_at_even_words(n, groups, cg):
    '''The rows' values, and behind them, from an even word on, mean and 1 / deviation of every row and group.'''
    forward, backward = norm_launches(n, 1, groups, cg)
    plan = K.norm_plan(n, 1, groups * cg, groups, False)
    assert plan.kind == 'rows'
    values, pairs = plan.M * plan.span, plan.M * plan.span // cg
    assert forward[0].lds == 4 * (values + values % 2 + 2 * pairs)
    #the gradient has two arrays of values in front of them: an even number of words
    plan = K.norm_plan(n, 1, groups * cg, groups, True)
    assert backward[0].lds == 4 * (2 * plan.M * plan.span + 4 * plan.M * plan.span // cg)


# ------------------------------------------------------------------ what the tests on the GPU reach

@pytest.mark.skipif(not (TOOLS and all(os.path.exists(build.hsaco_path(m)) for m in ('norm', 'recurrence'))), reason='no code object, or no tool to look into it')
def test_every_kernel_is_run_on_the_gpu(tmp_path):
    found = set(kernels_of('norm', tmp_path)) | set(kernels_of('recurrence', tmp_path))
    launched = {launch.kernel for size in NORM_SIZES for launches in norm_launches(*size) for launch in launches}
    launched |= {kernel for b, t, c in RECURRENCE_SIZES for gated in (False, True) for kernel in check_recurrence(b, t, c, gated, b > 1)}
    assert found == launched, (found - launched, launched - found)


# ------------------------------------------------------------------ results that are stored past the caches

@pytest.mark.parametrize('read', ['dfactor', 'dx', 'both', 'neither'])
def test_a_recurrences_gradient_is_stored_past_the_caches_where_neither_result_is_read(read):
    '''One flag is about both results: those that a later launch reads stay with the caches.'''
    shape = (2, 4096, 2048)
    large, small = np.broadcast_to(f32(0), shape), np.zeros((2, 2048), f32)

    def f(factor, x, h, g, last):
        dfactor, dx, dstate = lax.linear_recurrence_grad(h, factor, x, None, None, g, last)
        #(a product that has to have its operand in memory)
        reads = lambda v: lax.linear_recurrence(v, x)[1]
        return (reads(dfactor) if read in ('dfactor', 'both') else dfactor), (reads(dx) if read in ('dx', 'both') else dx), dstate
    program = JaxprInterpreter(mj.make_jaxpr(f)(large, large, large, large, small), plan_only=True)
    launch, = [l for l in program.launches if l.kernel.startswith('recurrence_grad')]
    assert bool(np.frombuffer(launch.params, np.uint32)[0] >> 31) == (read == 'neither')


# ------------------------------------------------------------------ many rows

@pytest.mark.parametrize('rows,v,top', [(2**24, 20, 0), (2**24 + 3, 130, 5), (2**25, 10, 10), (2**26 - 8, 100, 0), (2**26 - 8, 1000, 5)])
def test_log_probs_of_many_rows_are_planned(rows, v, top):
    assert all(not name.startswith('log_probs_block') for name in check_log_probs(rows, v, top))


@pytest.mark.parametrize('rows,v,top', [(2**31, 1, 0), (2**26, 1000, 5), (2**24, 5000, 0), (2**24 + 1, 4092, 0)])
def test_log_probs_of_too_many_rows_are_refused(rows, v, top):
    with pytest.raises(NotImplementedError):
        list(check_log_probs(rows, v, top))


# ------------------------------------------------------------------ many single steps

@pytest.mark.parametrize('b,c', [(2**19 + 1, 1024), (2**20, 1024), (300000, 2049), (2**19 - 1, 1024), (1, 2**29 - 2048)])
def test_single_steps_of_two_gigabytes_and_more_are_planned(b, c):
    x, state = buffer(b, 1, c), buffer(b, c)
    zeroed = lambda n, use: buffer(n, dtype=np.uint32)
    for launch, in (K.linear_recurrence(x, state, x, x, state, None, True, False, zeroed), K.linear_recurrence_grad(x, x, state, x, x, x, state, None, x, state, True, False, zeroed)):
        _, T, C, cstrips, strips, tiles, _, _, log2_w, _ = np.frombuffer(launch.params, np.uint32).astype(np.int64)
        vec = 4 if '_v4' in launch.kernel else 1
        assert T == tiles == 1 and strips * C == b * c * cstrips and cstrips * (vec << log2_w) >= C and launch.grid[0] == strips
        assert 4 * ((256 >> log2_w) * int(launch.kernel.split('_l')[1].split('_')[0]) * C + (vec << log2_w)) < 2**31 and launch.grid[0] * 256 < 2**32


# ------------------------------------------------------------------ what a group norm's gradient needs beside its operands

@pytest.mark.parametrize('n,s,groups,cg', [(8192, 1, 1, 16384), (8192, 1, 1, 16388), (8192, 1, 1, 8195), (4096, 4, 1, 8192), (100000, 2, 1, 8193), (5000, 15, 1, 9000), (4096, 16, 1, 9000), (64, 3136, 32, 8),
                                           (3000, 1, 2, 40000)])
def test_the_sums_of_channels_take_less_than_the_samples(n, s, groups, cg):
    c, taken = groups * cg, []

    def scratch(shape, dtype=np.float32):
        taken.append(int(np.prod(shape)))
        return buffer(*shape, dtype=dtype)
    x, small, stats = buffer(n, s, c), buffer(c), buffer(n, groups)
    K.group_norm_grad(x, small, small, x, x, small, small, stats, stats, groups, 1e-5, None, scratch)
    assert sum(taken) <= max(n * s * c // 4, 2 * 1024 * c)


# ------------------------------------------------------------------ what recurrences keep from launch to launch

@pytest.mark.parametrize('two_lanes', [False, True])
def test_recurrences_that_share_their_tickets_agree_on_everything_that_counts_them(two_lanes):
    '''Launches with one array of tickets and words have one kernel, one grid and one tiling, and run on one lane.'''
    def f(a, b, c):
        outs = [lax.linear_recurrence(v, v, reverse=r)[0] for v in (a, b, c) for r in (False, True)]
        outs += [nn.gated_recurrence(v, v)[1] for v in (a, b, c)]
        return outs + [mj.grad(lambda v: mj.numpy.sum(nn.gated_recurrence(v, v)[0]))(v) for v in (a, b, c)]
    args = [np.zeros(shape, f32) for shape in ((2, 2000, 64), (2, 2001, 64), (4, 2000, 36))]
    program = JaxprInterpreter(mj.make_jaxpr(f)(*args), plan_only=True, two_lanes=two_lanes)
    sharing, lanes = {}, program.lane_plan.lane if two_lanes else [0] * len(program.launches)
    for launch, lane in zip(program.launches, lanes):
        if launch.kernel.startswith('recurrence') and launch.kernel.endswith('_chain'):
            chain, = (launch.buffers[i][0] for i in launch.scratch)
            same = (launch.kernel, launch.grid, bytes(launch.params[12:36]), lane)      #(strips, tiles, lines of tickets, their parts, lanes)
            assert sharing.setdefault(id(chain), same) == same
    assert len(sharing) >= 6
