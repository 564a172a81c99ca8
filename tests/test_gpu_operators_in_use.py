'''Group norm, log probabilities of tokens and linear recurrences as programs use them: captured and replayed, side by side on two streams,
several calls in flight, operands that other operations leave (slices, transposes, broadcasts, the same array twice), nothing at all, and
arrays whose offsets pass 31 and 32 bits. Bounds are those of the operators' own tests.'''
import numpy as np
import pytest

import vkjax_amd
from tests.test_gpu_operators import U, both, close, norm_bounds, norm_program, probs_program, recurrence_inputs, recurrence_program
from tests.test_operators import normal
from vkjax_amd import minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

pytestmark = pytest.mark.gpu
jnp, lax, nn = mj.numpy, mj.lax, mj.nn
f32 = np.float32


def same(a, b):
    a, b = mj.tree_leaves(a), mj.tree_leaves(b)
    assert len(a) == len(b)
    for k, (x, y) in enumerate(zip(a, b)):
        assert np.array_equal(np.asarray(x).reshape(np.shape(y)), y, equal_nan=True), k


def cases():
    '''(name, program, arguments) of each operator in the forms that use scratch: chunks, slices, tiles that hand on their state'''
    g, x = normal(1, 5, 70, 71, 64), normal(2, 5, 70, 71, 64)
    yield 'norm', norm_program(8, 'silu'), [x, normal(3, 64), normal(4, 64), g]
    z, t = normal(5, 4, 90001), np.array([3, -1, 90000, 17], np.int32)
    yield 'probs', probs_program(7), [z, t, normal(6, 4), normal(7, 4), normal(8, 4, 7)]
    #few strips and many, whole vectors and single channels, sequences that end early
    for b, t, c, lengths in ((1, 5000, 100, False), (9, 1500, 132, True), (20, 900, 33, True), (1, 1300, 1001, False)):
        arrays = recurrence_inputs(b, t, c, True, True, lengths, seed=c)
        yield f'recurrence {b} x {t} x {c}', recurrence_program(True, bool(b % 2), list(arrays)), list(arrays.values())


CASES = list(cases())


@pytest.mark.parametrize('name,f,args', CASES, ids=[c[0] for c in CASES])
def test_captured_and_replayed_with_other_work_between(name, f, args):
    expected = mj.tree_leaves(vkjax_amd.wrap(f, frontend='minijax')(*args))
    program = JaxprInterpreter(mj.make_jaxpr(f)(*args), graph=True)
    program.upload_inputs(*args)
    other = vkjax_amd.wrap(f, frontend='minijax')
    for n in (1, 2, 1, 3):
        program.replay(n)
        same(program.read_outputs(), expected)
        same(other(*args), expected)
    #other values of the same sizes, then the first ones again
    changed = [a * f32(0.5) if a.dtype == f32 else a for a in args]
    halved = other(*changed)
    program.upload_inputs(*changed)
    program.replay(1)
    same(program.read_outputs(), halved)
    program.upload_inputs(*args)
    program.replay(1)
    same(program.read_outputs(), expected)


@pytest.mark.parametrize('name,f,args', CASES, ids=[c[0] for c in CASES])
def test_two_at_once_on_two_streams(name, f, args):
    def twice(*a):
        return f(*a), f(*[v * f32(0.5) if v.dtype == f32 else v for v in a])
    expected = vkjax_amd.wrap(twice, frontend='minijax')(*args)
    same(expected[0], vkjax_amd.wrap(f, frontend='minijax')(*args))
    lanes = vkjax_amd.wrap(twice, frontend='minijax', two_lanes=True)
    for _ in range(4):
        same(lanes(*args), expected)


@pytest.mark.parametrize('name,f,args', CASES, ids=[c[0] for c in CASES])
def test_several_calls_in_flight(name, f, args):
    plain, fast = (vkjax_amd.wrap(f, frontend='minijax') for _ in range(2))
    tuples = [tuple(a * f32(1 + k) if a.dtype == f32 else a for a in args) for k in range(4)]
    expected = [plain(*t) for t in tuples]
    got = list(fast.stream(iter(tuples), in_flight=2))
    assert len(got) == len(expected)
    for a, b in zip(got, expected):
        same(a, b)


def test_only_the_gradients_and_only_the_statistics():
    #results that nobody reads
    x, scale, shift, g = normal(1, 3, 40, 40, 24), normal(2, 24), normal(3, 24), normal(4, 3, 40, 40, 24)
    whole = mj.tree_leaves(vkjax_amd.wrap(norm_program(4, 'silu'), frontend='minijax')(x, scale, shift, g))
    for k in range(4):
        same(vkjax_amd.wrap(lambda *a: norm_program(4, 'silu')(*a)[k], frontend='minijax')(x, scale, shift, g), [whole[k]])
    z, t = normal(5, 3, 70000), np.array([1, 2, 3], np.int32)
    f = vkjax_amd.wrap(probs_program(3), frontend='minijax')
    args = [z, t, normal(6, 3), normal(7, 3), normal(8, 3, 3)]
    whole = mj.tree_leaves(f(*args))
    for k in range(len(whole)):
        same(vkjax_amd.wrap(lambda *a: probs_program(3)(*a)[k], frontend='minijax')(*args), [whole[k]])
    arrays = recurrence_inputs(2, 700, 40, True, True, True)
    f = recurrence_program(True, False, list(arrays))
    whole = mj.tree_leaves(vkjax_amd.wrap(f, frontend='minijax')(*arrays.values()))
    for k in range(len(whole)):
        same(vkjax_amd.wrap(lambda *a: f(*a)[k], frontend='minijax')(*arrays.values()), [whole[k]])


def test_the_same_array_in_several_places():
    x = normal(1, 6, 20, 20, 16)
    s = (0.5 + np.random.default_rng(0).random(16)).astype(f32)
    got, expected, _ = both(lambda x, s: norm_program(4, 'silu')(x, s, s, x), x, s)
    for name, a, b, bound in zip(('y', 'dx', 'dscale', 'dshift'), got, expected, norm_bounds(x, s, s, x, 4, 1e-5, 'silu')):
        close(a, b, bound, name)
    a = (1 - 0.4 * np.random.default_rng(1).random((2, 600, 40))).astype(f32)
    once = vkjax_amd.wrap(lambda a: lax.linear_recurrence(a, a), frontend='minijax')(a)
    same(once, vkjax_amd.wrap(lambda a, b: lax.linear_recurrence(a, b), frontend='minijax')(a, a.copy()))
    #the same primal twice: each place has its own gradient
    def gradients(a, b, g, l):
        _, pullback = mj.vjp(lambda p, q: lax.linear_recurrence(p, q), a, b)
        return pullback((g, l))
    g, l = normal(2, 2, 600, 40), normal(3, 2, 40)
    same(vkjax_amd.wrap(lambda a, g, l: gradients(a, a, g, l), frontend='minijax')(a, g, l),
         vkjax_amd.wrap(gradients, frontend='minijax')(a, a.copy(), g, l))


@pytest.mark.parametrize('fuse', [True, False], ids=['fused', 'unfused'])
def test_operands_and_results_of_other_operations(fuse):
    '''Slices at odd offsets, transposes, broadcasts, joined arrays and elementwise results go in, slices of the results come out.'''
    def wrap(f):
        return vkjax_amd.wrap(f, frontend='minijax', fuse=fuse)
    wide, row = normal(1, 7, 9, 11, 15), normal(2, 15)

    def norm(wide, row):
        x = jnp.transpose(wide, (1, 0, 2, 3))[1:, 1:, :, 2:14] * np.float32(2) + np.float32(1)
        y, pullback = mj.vjp(lambda x, s, b: nn.group_norm(x, s, b, 3, activation='relu'), x, row[3:], jnp.broadcast_to(row[0], (12,)))
        dx, dscale, dshift = pullback(jnp.tanh(jnp.transpose(wide[:6, :8, :, 1:13], (1, 0, 2, 3))))
        return x, y, dx[2:, 1], dscale + dshift
    got = wrap(norm)(wide, row)
    x = np.ascontiguousarray(wide.transpose(1, 0, 2, 3)[1:, 1:, :, 2:14]) * f32(2) + f32(1)
    assert np.array_equal(got[0], x)
    scale, shift = row[3:].copy(), np.full(12, row[0], f32)
    g = np.tanh(wide[:6, :8, :, 1:13].transpose(1, 0, 2, 3).astype(np.float64)).astype(f32)
    alone = vkjax_amd.wrap(lambda *a: norm_program(3, 'relu')(*a), frontend='minijax')(x, scale, shift, np.ascontiguousarray(g))
    assert np.array_equal(got[1], alone[0])
    #the cotangent through the device's tanh: 4 u of values of at most 1, against the bounds of the gradient itself
    bounds = norm_bounds(x, scale, shift, g, 3, 1e-5, 'relu')
    close(got[2], alone[1][2:, 1], 16 * bounds[1][2:, 1] + 1e-6, 'dx')

    table = normal(3, 31, 450)
    ids = np.array([[4, 2, 399], [0, -1, 400], [17, 8, 398]], np.int32)

    def probs(table, ids):
        logits = jnp.reshape(table[3:12, 25:425], (3, 3, 400))
        lp, entropy, top, which = nn.token_log_probs(logits, jnp.transpose(ids) + np.int32(1), 4)
        return jnp.exp(lp)[1:], entropy[:, 2], top[..., 1:3], which[1]
    alone = vkjax_amd.wrap(lambda z, t: nn.token_log_probs(z, t, 4), frontend='minijax')(table[3:12, 25:425].reshape(3, 3, 400).copy(), np.ascontiguousarray(ids.T) + 1)
    got = wrap(probs)(table, ids)
    same(got[1:], (alone[1][:, 2], alone[2][..., 1:3], alone[3][1]))
    close(got[0], np.exp(alone[0][1:].astype(np.float64)), 8 * U)

    series = normal(4, 3, 50, 41)
    gate = normal(5, 41) + f32(2)

    def recurrence(series, gate):
        x = jnp.concatenate([series[:, 1::2, 1:], series[:, ::2, :40]], axis=1)
        h, last = nn.gated_recurrence(jnp.broadcast_to(gate[:40], (3, 50, 40)), x, x[:, 7], np.array([50, 0, 13], np.int32))
        return h[:, 5:9, 3:], last * np.float32(2)
    x = np.concatenate([series[:, 1::2, 1:], series[:, ::2, :40]], axis=1)
    alone = vkjax_amd.wrap(lambda g, x, s, l: nn.gated_recurrence(g, x, s, l), frontend='minijax')(
        np.ascontiguousarray(np.broadcast_to(gate[:40], (3, 50, 40))), x, x[:, 7].copy(), np.array([50, 0, 13], np.int32))
    same(wrap(recurrence)(series, gate), (alone[0][:, 5:9, 3:], alone[1] * f32(2)))


def test_arrays_of_the_host_in_any_form():
    #other orders of memory, types that become 32 bits, a strided view
    x = np.asfortranarray(normal(1, 4, 9, 9, 12).astype(np.float64))
    s, b = normal(2, 24)[::2], normal(3, 12).astype(np.float64)
    f = vkjax_amd.wrap(lambda x, s, b: nn.group_norm(x, s, b, 3), frontend='minijax')
    same(f(x, s, b), f(np.ascontiguousarray(x, f32), s.copy(), b.astype(f32)))
    z, t = normal(4, 500, 8).T, np.arange(8, dtype=np.int64)
    f = vkjax_amd.wrap(lambda z, t: nn.token_log_probs(z, t, 2), frontend='minijax')
    same(f(z, t), f(np.ascontiguousarray(z), t.astype(np.int32)))
    f = vkjax_amd.wrap(lambda g, x, l: nn.gated_recurrence(g, x, None, l), frontend='minijax')
    g, x, l = normal(5, 30, 2, 7).transpose(1, 0, 2), normal(6, 2, 7, 30).transpose(0, 2, 1), np.array([30, 11], np.int64)
    same(f(g, x, l), f(np.ascontiguousarray(g), np.ascontiguousarray(x), l.astype(np.int32)))


@pytest.mark.parametrize('shape', [(0, 4, 8), (3, 0, 8), (0, 8)])
def test_group_norm_of_nothing(shape):
    got, expected, _ = both(norm_program(2, 'relu'), np.zeros(shape, f32), np.ones(8, f32), np.ones(8, f32), np.zeros(shape, f32))
    same(got, expected)


@pytest.mark.parametrize('v', [5, 600, 5000, 100000])
def test_log_probs_of_no_rows(v):
    got, expected, _ = both(probs_program(3), np.zeros((0, v), f32), np.zeros(0, np.int32), np.zeros(0, f32), np.zeros(0, f32), np.zeros((0, 3), f32))
    same(got, expected)


@pytest.mark.parametrize('b,t,c', [(0, 4, 8), (3, 0, 8), (3, 4, 0)])
@pytest.mark.parametrize('state,lengths', [(True, True), (False, False), (True, False)])
def test_recurrence_of_nothing(b, t, c, state, lengths):
    arrays = dict(factor=np.zeros((b, t, c), f32), x=np.zeros((b, t, c), f32))
    if state:
        arrays['state'] = normal(1, b, c)
    if lengths:
        arrays['lengths'] = np.ones(b, np.int32)
    arrays.update(g=normal(2, b, t, c), g_last=normal(3, b, c))
    for reverse in (False, True):
        got, expected, _ = both(recurrence_program(True, reverse, list(arrays)), *arrays.values())
        same(got, expected)


def test_group_norm_with_the_largest_use_of_shared_memory():
    x, scale, shift, g = normal(1, 2100, 4096), normal(2, 4096), normal(3, 4096), normal(4, 2100, 4096)
    got, expected, _ = both(norm_program(1, None), x, scale, shift, g)
    for name, a, b, bound in zip(('y', 'dx', 'dscale', 'dshift'), got, expected, norm_bounds(x, scale, shift, g, 1, 1e-5, None)):
        close(a, b, bound, name)


# ------------------------------------------------------------------ arrays whose offsets pass 31 bits, and 32

def test_group_norm_of_a_sample_of_two_gigabytes():
    '''x[s, c] = a[s] b[c], 2.4 GB in a sample: of its results the last positions.'''
    s, c, groups = 600007, 1000, 4
    a, b = (1 + 0.5 * np.random.default_rng(1).random(s)).astype(f32), normal(2, c)

    def f(a, b, one):
        x = jnp.reshape(a, (1, s, 1)) * jnp.reshape(b, (1, 1, c))
        y, pullback = mj.vjp(lambda x: nn.group_norm(x, one, one, groups), x)
        dx, = pullback(jnp.broadcast_to(jnp.reshape(b, (1, 1, c)), (1, s, c)))
        return y[:, s - 5:], dx[:, s - 5:]
    y, dx = vkjax_amd.wrap(f, frontend='minijax')(a, b, np.ones(c, f32))
    a64, b64 = a.astype(np.float64), b.astype(np.float64).reshape(groups, -1)
    mean = a64.mean() * b64.mean(axis=1)
    second = (a64 ** 2).mean() * (b64 ** 2).mean(axis=1)
    rstd = 1 / np.sqrt(second - mean ** 2 + 1e-5)
    hat = (a64[-5:, None, None] * b64 - mean[:, None]) * rstd[:, None]
    #values of at most 8 standard deviations: sums of 64 additions in a row, and a chunk's 300 joined four times over
    close(y[0], (hat + 1).reshape(5, c), 400 * U * 8, 'y')
    #the sums over the group of g and g hat, g = b
    m1 = b64.mean(axis=1)
    m2 = ((a64.mean() * (b64 ** 2).mean(axis=1)) - mean * m1) * rstd
    close(dx[0], (rstd[:, None] * (b64 - m1[:, None] - hat * m2[:, None])).reshape(5, c), 2000 * U * 8, 'dx')


def test_log_probs_of_more_than_four_gigabytes():
    '''11000 rows of 100003 (4.4 GB): rows of zeros but for some, of which the last stand behind the 32nd bit.'''
    rows, v = 11000, 100003
    z = np.zeros((rows, v), f32)
    t = np.full(rows, -1, np.int32)
    some = np.array([0, 1, 5368, 5370, 10736, 10738, 10741, rows - 2, rows - 1])
    z[some] = normal(1, len(some), v)
    t[some] = np.arange(len(some)) * 11111 + 3
    got = vkjax_amd.wrap(lambda z, t: nn.token_log_probs(z, t, 3), frontend='minijax')(z, t)
    z64 = z[some].astype(np.float64)
    logp = z64 - (z64.max(1) + np.log(np.exp(z64 - z64.max(1, keepdims=True)).sum(1)))[:, None]
    #64 additions in a row, twice over, and the logarithm's and the difference's own roundings of values of at most 20
    bound = 160 * U + 6 * U * 20
    close(got[0][some], logp[np.arange(len(some)), t[some]], bound)
    close(got[1][some], -(np.exp(logp) * logp).sum(1), 20 * bound)
    order = np.argsort(-z64, axis=1, kind='stable')[:, :3]
    assert np.array_equal(got[3][some], order)
    close(got[2][some], np.take_along_axis(logp, order, 1), bound)
    padded = np.setdiff1d(np.arange(rows), some)
    assert not got[0][padded].any() and not got[1][padded].any() and not got[2][padded].any() and (got[3][padded] == -1).all()


def test_log_probs_gradient_of_three_gigabytes():
    rows, v = 8001, 100003
    row, t = normal(1, v), ((np.arange(8001) * 12345) % 100003).astype(np.int32)

    def f(row, t):
        z = jnp.broadcast_to(jnp.reshape(row, (1, v)), (rows, v))
        lp, pullback = mj.vjp(lambda z: nn.token_log_probs(z, t)[0], z)
        dz, = pullback(lp * np.float32(0) + np.float32(1))
        return lp, dz[rows - 3:]
    lp, dz = vkjax_amd.wrap(f, frontend='minijax')(row, t)
    r = row.astype(np.float64)
    logp = r - (r.max() + np.log(np.exp(r - r.max()).sum()))
    close(lp, logp[t], 160 * U + 6 * U * 20)
    expected = -np.exp(logp)[None].repeat(3, 0)
    expected[np.arange(3), t[-3:]] += 1
    close(dz, expected, (160 + 120) * U * np.abs(expected) + 4 * U * (np.abs(expected) > 0.5))


@pytest.mark.parametrize('b,t,c', [(1, 430001, 1252), (430001, 5, 256)])
def test_recurrence_of_two_gigabytes(b, t, c):
    '''The same gates at every time, and an addend that depends on it: the last times of the last sequence.'''
    gate, x = normal(1, c) + f32(1), normal(2, t)

    def f(gate, x):
        gates = jnp.broadcast_to(jnp.reshape(gate, (1, 1, c)), (b, t, c))
        xs = jnp.broadcast_to(jnp.reshape(x, (1, t, 1)), (b, t, c))
        (h, last), pullback = mj.vjp(lambda g, x: nn.gated_recurrence(g, x), gates, xs)
        _, dx = pullback((xs, jnp.zeros((b, c), np.float32)))
        return h[b - 1, t - 5:], last[b - 1], dx[b - 1, t - 5:]
    h, last, dx = vkjax_amd.wrap(f, frontend='minijax')(gate, x)
    a = 1 / (1 + np.exp(-gate.astype(np.float64)))
    now, times = np.zeros(c), []
    for k in range(t):
        now = a * now + (1 - a) * float(x[k])
        if k >= t - 5:
            times.append(now)
    #24 u of values of at most 6 at every step, of which a stay: 1 / (1 - a) of them
    bound = 24 * U * 6 / (1 - a)
    close(h, np.array(times), bound)
    close(last, now, bound)
    l, ls = np.zeros(c), []
    for k in range(t - 1, t - 6, -1):
        l = float(x[k]) + a * l
        ls.append(l * (1 - a))
    close(dx, np.array(ls[::-1]), 48 * U * 6 * 5)


# ------------------------------------------------------------------ many alternatives, of which more stand out at once than there is room for

@pytest.mark.parametrize('rows,v,levels', [(600, 167, None), (300, 511, 40), (500, 1000, None), (400, 4092, None), (200, 8000, 300), (150, 22133, None), (3, 127677, None),
                                           (2, 127677, 7), (2, 100000, 1), (900, 19, 3), (64, 129, 2)])
@pytest.mark.parametrize('top', [19, 24, 32])
def test_many_alternatives(rows, v, levels, top):
    '''Scores of any value, or of few different ones: which are alternatives, and in what order, is exact.'''
    top = min(top, v)
    rng = np.random.default_rng(rows + v + top)
    z = normal(rows + v, rows, v, scale=2.0) if levels is None else rng.integers(0, levels, (rows, v)).astype(f32)
    z[rng.random((rows, v)) < 0.3 * (np.arange(rows) % 3 == 0)[:, None]] = -np.inf
    t = rng.integers(0, v, rows).astype(np.int32)
    log_p, _, top_log_p, tokens = vkjax_amd.wrap(lambda z, t: nn.token_log_probs(z, t, top), frontend='minijax')(z, t)
    order = np.argsort(-z, axis=1, kind='stable')[:, :top]
    assert np.array_equal(tokens, order)
    z64 = z.astype(np.float64)
    most = z64.max(1)
    logp = z64 - np.where(most == -np.inf, 0.0, most + np.log(np.exp(z64 - np.where(most == -np.inf, 0.0, most)[:, None]).sum(1)))[:, None]
    #sums of up to 64 additions in a row, joined four times over, and roundings of values of at most 30 (and 300)
    bound = (64 + 16) * 2 * U + 6 * U * (30 if levels is None else 300 + 12)
    close(top_log_p, np.take_along_axis(logp, order, 1), bound)
    close(log_p, logp[np.arange(rows), t], bound)


@pytest.mark.parametrize('n,c,groups', [(1, 1194, 1), (3, 2049, 1), (700, 1194, 1), (2100, 8192, 1), (5, 16384, 2), (2, 16384, 1), (1, 20000, 1), (9, 6141, 3), (1300, 4100, 1), (3, 32772, 1),
                                        (4, 8193, 1)])
@pytest.mark.parametrize('activation', [None, 'silu'])
def test_layer_norm_of_wide_rows(n, c, groups, activation):
    x, scale, shift, g = (normal(n + c, n, c) + normal(2, c)).astype(f32), normal(3, c), normal(4, c), normal(5, n, c)
    got, expected, _ = both(norm_program(groups, activation), x, scale, shift, g)
    for name, a, b, bound in zip(('y', 'dx', 'dscale', 'dshift'), got, expected, norm_bounds(x, scale, shift, g, groups, 1e-5, activation)):
        close(a, b, bound, name)


@pytest.mark.parametrize('shape,groups', [((1, 80, 80, 96), 12), ((1, 70, 70, 320), 32), ((1, 60, 61, 200), 25), ((2, 49, 72, 448), 64), ((1, 130, 127, 36), 9), ((3, 90, 41, 100), 4),
                                          ((1, 5000, 1100), 1), ((2, 4000, 66), 66)])
def test_group_norm_in_spans_of_few_groups(shape, groups):
    c = shape[-1]
    x, scale, shift, g = (normal(c, *shape) + normal(2, c)).astype(f32), normal(3, c), normal(4, c), normal(5, *shape)
    got, expected, _ = both(norm_program(groups, 'silu'), x, scale, shift, g)
    for name, a, b, bound in zip(('y', 'dx', 'dscale', 'dshift'), got, expected, norm_bounds(x, scale, shift, g, groups, 1e-5, 'silu')):
        close(a, b, bound, name)


@pytest.mark.parametrize('name,f,args', CASES, ids=[c[0] for c in CASES])
def test_profiled_and_with_every_value_returned(name, f, args):
    expected = mj.tree_leaves(vkjax_amd.wrap(f, frontend='minijax')(*args))
    outs, info = vkjax_amd.wrap(f, frontend='minijax', profiling=True)(*args)
    same(outs, expected)
    assert info
    closed = mj.make_jaxpr(f)(*args)
    outs, values = JaxprInterpreter(closed, reuse_buffers=False).run(*args, return_all=True)
    same(outs, expected)
    #every result of the operators' equations that something reads
    results = [v for eqn in closed.jaxpr.eqns if eqn.primitive.name in ('group_norm', 'token_log_probs', 'linear_recurrence') for v in eqn.outvars]
    assert results and all(np.isfinite(np.asarray(values[v], np.float64)).any() for v in results if v in values)
