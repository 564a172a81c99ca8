'''How launches of group norms, log probabilities and recurrences are cut, over the ranges of sizes that they take: every element has a
lane, shared memory suffices, and the kernels that are chosen exist.'''
import os
import random
import re
import shutil
import subprocess

import numpy as np
import pytest

from vkjax_amd import kernels as K
from vkjax_amd.buffers import Buffer
from vkjax_amd.csrc import build

LLVM = '/opt/rocm/llvm/bin'
TOOLS = all(shutil.which(f'{LLVM}/{t}') for t in ('clang-offload-bundler', 'llvm-readelf'))


def kernels_of(module, tmp_path):
    '''{kernel: (vector registers, bytes of scratch memory)}'''
    obj = str(tmp_path / f'{module}.o')
    subprocess.run([f'{LLVM}/clang-offload-bundler', '--unbundle', '--type=o', '--targets=hipv4-amdgcn-amd-amdhsa--gfx950',
                    f'--input={build.hsaco_path(module)}', f'--output={obj}'], check=True)
    notes = subprocess.run([f'{LLVM}/llvm-readelf', '--notes', obj], check=True, capture_output=True, text=True).stdout
    field = lambda k, name: re.search(rf'\.{name}:\s+(\S+)', k).group(1)
    return {field(k, 'name'): (int(field(k, 'vgpr_count')), int(field(k, 'private_segment_fixed_size'))) for k in notes.split('- .agpr_count')[1:]}


def words(launch):
    return np.frombuffer(launch.params, np.uint32).astype(np.int64)


def buffer(*shape, dtype=np.float32):
    return Buffer(None, np.dtype(dtype), shape)


def scratch(shape, dtype=np.float32):
    return buffer(*shape, dtype=dtype)


def log_int(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def norm_launches(n, s, groups, cg, activation='silu'):
    c = groups * cg
    x, small, stats = buffer(n, s, c), buffer(c), buffer(n, groups)
    forward  = K.group_norm(x, stats, stats, x, small, small, groups, 1e-5, activation, scratch)
    backward = K.group_norm_grad(x, small, small, x, x, small, small, stats, stats, groups, 1e-5, activation, scratch)
    return forward, backward


def check_norm(n, s, groups, cg):
    c = groups * cg
    for gradient, launches in enumerate(norm_launches(n, s, groups, cg)):
        for launch in launches:
            assert launch.grid[0] * launch.block[0] < 2**32
            if launch.kernel == 'group_norm_columns':
                yield launch.kernel
                continue
            _, N, S, C, G, CG, _, _, span, spans, pieces, V, P, M, lc, lq, chunks, chunk = words(launch)[:18]
            plan = K.norm_plan(n, s, c, groups, bool(gradient))
            assert (N, S, C, G, CG) == (n, s, c, groups, cg)
            threads = launch.block[0]
            vec = plan.vec
            assert span % vec == 0 and V == span // vec and lc + lq <= 6
            if pieces == 1:
                assert span % cg == 0 and spans * span >= c > (spans - 1) * span
            else:
                assert pieces * span >= cg > (pieces - 1) * span and spans == groups * pieces and (vec == 1 or cg % 4 == 0)
            per_group = max(span // cg, 1)
            room = launch.lds // 4
            if plan.kind == 'wide':
                assert s == 1 and span == cg and spans == groups and cg % vec == 0 and plan.k * threads * vec >= cg and launch.lds == 0
                assert launch.grid[0] % groups == 0 and (gradient or launch.grid[0] == n * groups)
            elif plan.kind == 'held':
                assert V * P * M <= threads and P * plan.k >= s and P <= s
                assert room >= 2 * M * P * span + 2 * per_group * M and M * s * c * 4 < 2**31
            elif plan.kind == 'rows':
                assert s == 1 and P == 1 and V * (M // plan.k) <= threads and M % plan.k == 0 and (vec == 1 or cg > 1)
                assert room >= (2 * M * span + 4 * per_group * M if gradient else M * span + 2 * per_group * M) and M * c * 4 < 2**31
            else:
                assert V * P <= threads and chunks * chunk >= s > (chunks - 1) * chunk and chunk * c * 4 < 2**31
                assert room >= (2 * P * span if 'stats' in launch.kernel or 'sums' in launch.kernel else 2 * per_group)
                assert launch.grid[0] == n * chunks * spans
            #a CU's 160 KB hold two blocks of the largest
            assert launch.lds <= 80 << 10
            yield launch.kernel


def check_log_probs(rows, v, top):
    z, t = buffer(rows, v), buffer(rows, dtype=np.int32)
    r, k = buffer(rows), buffer(rows, top)
    launches = K.token_log_probs(r, r, r, k if top else None, k if top else None, z, t, top, scratch)
    vectors = -(-(v + (3 if v % 4 else 0)) // 4)
    for launch in launches:
        assert launch.grid[0] * launch.block[0] < 2**32 and launch.lds <= 64 << 10
        _, R, V, T, slices, slice_, log2_lanes = words(launch)
        assert (R, V, T) == (rows, v, top)
        if launch.kernel == 'log_probs_short':
            assert 4 << log2_lanes >= vectors and log2_lanes <= 6 and launch.grid[0] * 256 >= rows << log2_lanes
        elif launch.kernel.startswith('log_probs_wave'):
            assert launch.grid[0] * 4 >= rows and (launch.kernel != 'log_probs_wave' or vectors <= 256)
        elif launch.kernel == 'log_probs_block':
            assert slices * 4 * slice_ >= vectors and slice_ % 64 == 0 and launch.grid[0] == rows * slices
        else:
            assert slices * top <= 1024 and launch.lds == 0
        yield launch.kernel
    launch, = K.token_log_probs_grad(z, z, t, r, r, r, r, k if top else None, k if top else None, top)
    rows_, R, V, T, slices, slice_, log2_lanes = words(launch)
    assert rows_ == rows and slices * slice_ >= vectors and slice_ % 4 == 0 and launch.grid[0] >= -(-rows // (256 >> log2_lanes)) * slices
    #a block's scores lie within what a descriptor addresses
    assert ((256 >> log2_lanes) * v + 3) * 4 < 2**31 and launch.grid[0] * 256 < 2**32
    yield launch.kernel


def check_recurrence(b, t, c, gated=True, lengths=True):
    x, state = buffer(b, t, c), buffer(b, c)
    zeroed = lambda n, use: buffer(n, dtype=np.uint32)
    args = (x, x, state, buffer(b, dtype=np.int32) if lengths else None)
    for launch, in (K.linear_recurrence(x, state, *args, gated, False, zeroed), K.linear_recurrence_grad(x, x, state, x, *args, x, state, gated, True, zeroed)):
        _, T, C, cstrips, strips, tiles, lines, of_each, log2_w, _ = words(launch)
        vec, steps = (int(n) for n in re.search(r'_v(\d)_l(\d+)', launch.kernel).groups())
        W, G = 1 << log2_w, 256 >> log2_w
        assert (T, C) in ([(t, c), (1, b * c)] if t == 1 and not lengths else [(t, c)]) and (vec == 1 or C % 4 == 0)
        assert cstrips * W * vec >= C > (cstrips - 1) * W * vec and strips == b * c // C * cstrips and tiles * G * steps >= T > (tiles - 1) * G * steps
        assert (G * steps * C + W * vec) * 4 < 2**31 and launch.grid[0] * 256 < 2**32
        chain = launch.buffers[-1][0]
        if tiles == 1:
            assert chain is None and launch.grid[0] == strips and not launch.scratch
        else:
            #the words of every tile and channel behind the tickets' lines; 32 channels at most; a block for every tile of every line of tickets
            assert W * vec <= K.RECURRENCE_CHAIN_CHANNELS and chain.size >= 2 * (8 * K.RECURRENCE_LINES + tiles * strips * W * vec)
            every = cstrips if of_each else strips
            mine = [strips // every * (every * (i + 1) // lines - every * i // lines) for i in range(lines)]
            assert lines in (1, 8)
            assert launch.grid[0] % lines == 0 and launch.grid[0] // lines >= max(mine) * tiles and min(mine) > 0 and sum(mine) == strips
            assert launch.scratch == (len(launch.buffers) - 1,) and launch.scratch[0] in launch.written
        yield launch.kernel


def everything():
    rng, names = random.Random(5), set()
    for n, s, groups, cg in ([(1, 1, 1, 1), (1, 49, 32, 16), (32, 3136, 32, 2), (64, 3136, 32, 8), (8191, 1, 16, 65), (5, 1, 1, 8191), (100, 1, 1, 8192), (2, 12, 5, 1001), (3, 7, 1, 4100),
                              (70000, 1, 1, 4), (1, 1 << 20, 4, 16), (2, 5, 1024, 1), (9, 4, 3, 1), (4096, 1, 1, 4096), (7, 1, 1, 1023), (300, 2, 2, 6), (64, 3, 2, 2044), (300, 1, 1, 8192), (300, 1, 2, 16380), (17, 1, 1, 32768), (300, 1, 1, 1194), (9, 1, 3, 2047), (5, 1, 1, 40000)]
                             + [(log_int(rng, 1, 4096), log_int(rng, 1, 12544), rng.choice((1, 2, 3, 8, 32)), log_int(rng, 1, 300)) for _ in range(300)]
                             + [(log_int(rng, 1, 20000), 1, rng.choice((1, 2, 3, 8, 16, 64)), log_int(rng, 1, 3000)) for _ in range(150)]):
        names.update(check_norm(n, s, groups, cg))
    for rows, v, top in ([(1, 1, 0), (65536, 10, 10), (1, 500000, 32), (4096, 32000, 0), (1023, 4097, 20), (1024, 4096, 20), (1 << 20, 128, 1), (3, 100003, 1)]
                         + [(log_int(rng, 1, 65536), log_int(rng, 1, 300000), rng.choice((0, 1, 5, 20, 32))) for _ in range(300)]):
        names.update(check_log_probs(rows, v, min(top, v)))
    for b, t, c in ([(1, 1, 1), (64, 1, 2048), (1, 65536, 1024), (8, 2048, 2048), (3, 1021, 333), (70000, 2, 4), (1, 1 << 20, 1), (2, 17, 1 << 18)]
                    + [(log_int(rng, 1, 300), log_int(rng, 1, 70000), log_int(rng, 1, 5000)) for _ in range(300)]):
        for gated in (False, True):
            names.update(check_recurrence(b, t, c, gated, rng.random() < 0.5))
    return names


def test_launches_cover_their_operands():
    everything()


@pytest.mark.skipif(not (TOOLS and all(os.path.exists(build.hsaco_path(m)) for m in ('norm', 'log_probs', 'recurrence'))), reason='no code object, or no tool to look into it')
def test_kernels_exist_and_keep_their_registers(tmp_path):
    found = {}
    for module in ('norm', 'log_probs', 'recurrence'):
        found.update(kernels_of(module, tmp_path))
    names = everything()
    assert names <= set(found), names - set(found)
    #every kernel is one that some size reaches, none keeps registers in memory, and a block of 256 threads fits a SIMD twice
    assert set(found) == names, set(found) - names
    assert all(scratch_ == 0 and vgprs <= 256 for vgprs, scratch_ in found.values()), {k: v for k, v in found.items() if v[1] or v[0] > 256}


def test_sizes_that_are_refused():
    with pytest.raises(NotImplementedError):
        list(check_log_probs(1, 1 << 29, 0))
    with pytest.raises(NotImplementedError):
        list(check_recurrence(1, 4, 1 << 28))
    with pytest.raises(NotImplementedError):
        norm_launches(1 << 27, 1, 1, 1024)
