'''Short causal convolutions, selective scans, log probabilities from weights and orthogonalised updates as programs use them: one token model that is trained and that answers token by token,
captured and replayed, side by side on two streams, several calls in flight, operands that other operations leave, and arrays whose offsets pass 31 and 32 bits. Bounds are those of the
operators' own tests.'''
import numpy as np
import pytest

import vkjax_amd
from tests.test_gpu_operators import U, both, close
from tests.test_gpu_operators_in_use import same
from tests.test_gpu_token_model_operators import conv_bounds, conv_program, loss_bounds, loss_inputs, orthogonal_bound, scan_bounds
from tests.test_operators import normal
from tests.test_token_model_operators import OPTIONAL, loss_program, scan_inputs, scan_program
from oracle import primitives as P
from oracle.eval_jaxpr import eval_closed_jaxpr
from vkjax_amd import kernels as K, minijax as mj
from vkjax_amd.jaxpr_interpreter import JaxprInterpreter

pytestmark = pytest.mark.gpu
jnp, lax, nn = mj.numpy, mj.lax, mj.nn
f32 = np.float32
DEFAULT = (3.4445, -4.7750, 2.0315)


def wrap(f, **kwargs):
    return vkjax_amd.wrap(f, frontend='minijax', **kwargs)


# ------------------------------------------------------------------ a token model

def token_model(channels, inner, states, vocabulary, width, seed=0):
    '''Parameters: an embedding that is the output's weights too, and one layer.'''
    rng = np.random.default_rng(seed)
    draw = lambda *s, scale=1.0: (scale * rng.standard_normal(s)).astype(f32)
    return dict(table=draw(vocabulary, channels, scale=channels ** -0.5), into=draw(channels, 2 * inner, scale=channels ** -0.5), kernel=draw(width, inner, scale=0.5), bias=draw(inner, scale=0.1),
                step=draw(inner, inner, scale=inner ** -0.5), step_bias=(draw(inner) - 3).astype(f32), maps=draw(inner, 2 * states, scale=inner ** -0.5),
                decay=np.log(np.tile(np.arange(1, states + 1, dtype=f32), (inner, 1))), through=np.ones(inner, f32), back=draw(inner, channels, scale=inner ** -0.5))


def times(x, w):
    return jnp.reshape(jnp.dot(jnp.reshape(x, (-1, x.shape[-1])), w), tuple(x.shape[:-1]) + (w.shape[-1],))


def hidden(p, ids, states=(None, None), lengths=None):
    '''The layer's outputs for tokens [batch, time], and where it stands behind them.'''
    x = p['table'][ids]
    inner, n = p['kernel'].shape[1], p['decay'].shape[1]
    u = times(x, p['into'])
    u, gate = u[..., :inner], u[..., inner:]
    u, rows = nn.causal_conv(u, p['kernel'], p['bias'], states[0], lengths, 'silu')
    maps = times(u, p['maps'])
    y, held = nn.selective_scan(u, times(u, p['step']), -jnp.exp(p['decay']), maps[..., :n], maps[..., n:], p['through'], gate, states[1], lengths, p['step_bias'], True)
    return x + times(y, p['back']), (rows, held)


def loss(p, ids, lengths, targets, count):
    x, _ = hidden(p, ids, lengths=lengths)
    log_probs, _ = nn.linear_log_probs(x, p['table'], targets, transposed=True)
    return -jnp.sum(log_probs) / count


def batch_of(batch, time, vocabulary, lengths, seed=3):
    ids = np.random.default_rng(seed).integers(0, vocabulary, (batch, time + 1)).astype(np.int32)
    inside = np.arange(time)[None] < np.asarray(lengths)[:, None]
    return ids[:, :-1].copy(), np.where(inside, ids[:, 1:], -1).astype(np.int32), f32(inside.sum())


def train_step(p, momenta, ids, lengths, targets, count):
    '''Matrices are moved along their orthogonalised momentum, everything else along its gradient.'''
    value, grads = mj.value_and_grad(lambda p: loss(p, ids, lengths, targets, count))(p)
    moved, kept = {}, {}
    for k, v in p.items():
        if k in momenta:
            kept[k] = np.float32(0.9) * momenta[k] + grads[k]
            moved[k] = v - np.float32(0.02) * nn.orthogonalize(kept[k])
        else:
            moved[k] = v - np.float32(0.1) * grads[k]
    return value, moved, kept, grads


SIZES = [dict(channels=40, inner=72, states=8, vocabulary=203, width=4), dict(channels=24, inner=33, states=5, vocabulary=1001, width=3)]


@pytest.mark.parametrize('sizes', SIZES, ids=str)
@pytest.mark.parametrize('time', [9, 150])
def test_a_training_step_of_a_token_model(sizes, time):
    '''The gradient against the one that 64-bit steps give, and against differences of the loss; updates against those of their gradients.'''
    p = token_model(**sizes)
    lengths = np.array([time, 1, time // 2, 0], np.int32)
    ids, targets, count = batch_of(4, time, sizes['vocabulary'], lengths)
    momenta = {k: normal(i, *p[k].shape, scale=1e-3) for i, k in enumerate(('into', 'step', 'maps', 'back'))}
    step = wrap(lambda p, m, ids, lengths, targets: train_step(p, m, ids, lengths, targets, count))
    value, moved, kept, grads = step(p, momenta, ids, lengths, targets)
    program = mj.make_jaxpr(lambda p: mj.value_and_grad(lambda p: loss(p, ids, lengths, targets, count))(p))(p)
    names = sorted(p)
    expected = dict(zip(['value'] + names, eval_closed_jaxpr(program, *mj.tree_leaves(p))))
    #some twenty operations one behind the other, each off by at most 64 u of numbers that are ten times as large as its results at most
    close(value, expected['value'], 20 * 64 * 10 * U * abs(float(expected['value'])))
    for k in names:
        close(grads[k], expected[k], 20 * 64 * 10 * U * np.abs(expected[k]).max() + 1e-12, k)

    #along the gradient: the loss at either side, whose own error is that of 20 operations again; what the difference leaves out goes with the square of the distance
    direction = {k: (grads[k] / np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads.values()))).astype(f32) for k in names}
    evaluate = wrap(lambda p, ids, lengths, targets: loss(p, ids, lengths, targets, count))
    along = lambda e: (float(evaluate({k: p[k] + f32(e) * direction[k] for k in names}, ids, lengths, targets))
                       - float(evaluate({k: p[k] - f32(e) * direction[k] for k in names}, ids, lengths, targets))) / (2 * e)
    slope = sum((grads[k].astype(np.float64) * direction[k]).sum() for k in names)
    wide, near = along(0.04), along(0.02)
    rounding = 64 * U * abs(float(value)) / 0.02
    assert abs(near - slope) <= abs(wide - near) + 2 * rounding, (near, wide, slope, rounding)

    #updates: bit by bit those of the same operations by themselves
    for k in names:
        if k in momenta:
            m = wrap(lambda m, g: np.float32(0.9) * m + g)(momenta[k], grads[k])
            assert np.array_equal(kept[k], m), k
            assert np.array_equal(moved[k], wrap(lambda v, m: v - np.float32(0.02) * nn.orthogonalize(m))(p[k], m)), k
            x = m.astype(f32)
            off = (p[k].astype(np.float64) - moved[k]) / 0.02
            #(the step is rounded with the weight: half a unit of weights up to 4 over 0.02, per element)
            assert np.linalg.norm(off - P.orthogonalize(x, 5, DEFAULT, 1e-7)) <= orthogonal_bound(x, 5, DEFAULT) + 4 * U / 0.02 * np.sqrt(x.size), k


@pytest.mark.parametrize('sizes', SIZES, ids=str)
def test_token_by_token_as_the_prompt(sizes):
    '''Sequences of different lengths: behind their prompts (all at once, or a part and the rest) they stand where they are when every token came by itself, and tokens' log probabilities agree.'''
    p = token_model(**sizes)
    time, lengths = 37, np.array([37, 0, 20, 1, 36], np.int32)
    ids, targets, _ = batch_of(5, time, sizes['vocabulary'], lengths)

    def answer(p, ids, targets, lengths, rows, held):
        x, states = hidden(p, ids, (rows, held), lengths)
        return nn.linear_log_probs(x, p['table'], targets, transposed=True)[0], states
    f = wrap(answer)
    start = np.zeros((5, sizes['width'] - 1, sizes['inner']), f32), np.zeros((5, sizes['inner'], sizes['states']), f32)
    whole, end = f(p, ids, targets, lengths, *start)
    states, single = start, []
    for t in range(time):
        lp, states = f(p, ids[:, t:t + 1], targets[:, t:t + 1], (lengths > t).astype(np.int32), *states)
        single.append(lp[:, 0])
    first, middle = f(p, ids[:, :20], targets[:, :20], np.minimum(lengths, 20), *start)
    second, parted = f(p, ids[:, 20:], targets[:, 20:], np.maximum(lengths - 20, 0), *middle)
    #(as above: some twelve operations, off by 64 u of ten times their results)
    bound = 12 * 64 * 10 * U
    for a in (np.stack(single, 1), np.concatenate([first, second], 1)):
        close(a, whole, bound * np.abs(whole).max())
    for a, b, c in zip(states, parted, end):
        close(a, c, bound * np.abs(c).max())
        close(b, c, bound * np.abs(c).max())
    assert not whole[1].any() and not whole[2, 20:].any()


def test_a_training_step_captured_and_replayed():
    sizes = SIZES[0]
    p = token_model(**sizes)
    lengths = np.array([64, 30, 1], np.int32)
    ids, targets, count = batch_of(3, 64, sizes['vocabulary'], lengths)
    momenta = {k: normal(i, *p[k].shape, scale=1e-3) for i, k in enumerate(('into', 'step', 'maps', 'back'))}
    f = lambda p, m, ids, lengths, targets: train_step(p, m, ids, lengths, targets, count)
    eager = wrap(f)
    args = (p, momenta, ids, lengths, targets)
    names = sorted(p)

    def check(outs, expected):
        value, moved, kept, grads = expected
        parts = [[np.float32(0)], names, sorted(kept), names]
        outs, flat = list(mj.tree_leaves(outs)), list(mj.tree_leaves(expected))
        assert len(outs) == len(flat) == sum(len(v) for v in parts)
        for label, a, b in zip(['value'] + [f'moved {k}' for k in names] + [f'kept {k}' for k in sorted(kept)] + [f'gradient {k}' for k in names], outs, flat):
            a = np.asarray(a).reshape(np.shape(b))
            if label.endswith('table'):
                #a token's rows are added up as they arrive: at most 192 of them
                close(a, b, 2 * 192 * U * np.abs(grads['table']).max() + 2 * U * np.abs(b), label)
            else:
                assert np.array_equal(a, b), label
    expected = eager(*args)
    program = JaxprInterpreter(mj.make_jaxpr(f)(*args), graph=True)
    program.upload_inputs(*mj.tree_leaves(args))
    for n in (1, 2, 1, 3):
        program.replay(n)
        check(program.read_outputs(), expected)
        check(eager(*args), expected)


# ------------------------------------------------------------------ each by itself

def cases():
    '''(name, program, arguments) of each operator in the forms that use scratch: chunks of time, sums over blocks, shared contractions, kept scores'''
    x, kernel = normal(1, 5, 700, 132), normal(2, 4, 132)
    yield 'conv', conv_program(np.array([700, 0, 3, 650, 1], np.int32), 'silu', True, True), [x, kernel, normal(3, 5, 700, 132), normal(4, 5, 3, 132), normal(5, 132), normal(6, 5, 3, 132)]
    for b, t, c, n, given, lengths in ((1, 3000, 100, 16, OPTIONAL, None), (3, 500, 70, 5, ('gate',), np.array([500, 7, 0], np.int32)), (64, 1, 100, 16, ('state', 'd'), None)):
        arrays, g, g_last = scan_inputs(b, t, c, n, given, True)
        yield f'scan {b} x {t} x {c}', scan_program(list(arrays), lengths, True), [g, g_last, *arrays.values()]
    for rows, h, v, transposed in ((40, 200, 3001, False), (64, 130, 900, True), (142, 1500, 1100, False), (300, 70, 5003, True)):
        w = loss_inputs(rows, h, v, transposed)
        yield f'loss {rows} x {h} x {v}', loss_program(transposed), list(w)
    yield 'orthogonal', lambda x: (nn.orthogonalize(x, 3),), [normal(7, 3, 200, 900)]
    yield 'orthogonal tall', lambda x: (nn.orthogonalize(x, 2),), [normal(8, 1500, 333)]
    yield 'orthogonal of few rows', lambda x: (nn.orthogonalize(x),), [normal(9, 5, 50, 700)]
    yield 'orthogonal of few columns', lambda x: (nn.orthogonalize(x),), [normal(10, 3, 2000, 21)]
    yield 'conv of single steps', conv_program(None, 'silu', True, True), [normal(i, *s) for i, s in enumerate(((9, 1, 132), (4, 132), (9, 1, 132), (9, 3, 132), (132,), (9, 3, 132)))]
    yield 'loss of many features', loss_program(True), list(loss_inputs(7, 2100, 17003, True))


CASES = list(cases())
each = pytest.mark.parametrize('name,f,args', CASES, ids=[c[0] for c in CASES])


def test_the_cases_share_contractions():
    names = set()
    for _, f, args in CASES:
        program = JaxprInterpreter(mj.make_jaxpr(f)(*args))
        names |= {launch.kernel for launch in program.launches if launch is not None}
    assert any(n.startswith('linear_scores') and n.endswith('_shared') for n in names) and any(n.startswith('orthogonal') and n.endswith('_shared') for n in names), sorted(names)


@each
def test_captured_and_replayed_with_other_work_between(name, f, args):
    expected = mj.tree_leaves(wrap(f)(*args))
    program = JaxprInterpreter(mj.make_jaxpr(f)(*args), graph=True)
    program.upload_inputs(*args)
    other = wrap(f)
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


@each
def test_two_graphs_of_one_program_in_turn(name, f, args):
    programs = [JaxprInterpreter(mj.make_jaxpr(f)(*args), graph=True) for _ in range(2)]
    halves = [args, [a * f32(0.5) if a.dtype == f32 else a for a in args]]
    expected = [mj.tree_leaves(wrap(f)(*a)) for a in halves]
    for p, a in zip(programs, halves):
        p.upload_inputs(*a)
    for _ in range(3):
        for p in programs:
            p.replay(2)
    for p, e in zip(programs, expected):
        same(p.read_outputs(), e)


@each
def test_two_at_once_on_two_streams(name, f, args):
    def twice(*a):
        return f(*a), f(*[v * f32(0.5) if v.dtype == f32 else v for v in a])
    expected = wrap(twice)(*args)
    same(expected[0], wrap(f)(*args))
    lanes = wrap(twice, two_lanes=True)
    for _ in range(4):
        same(lanes(*args), expected)


@each
def test_several_calls_in_flight(name, f, args):
    plain, fast = (wrap(f) for _ in range(2))
    tuples = [tuple(a * f32(1 + k) if a.dtype == f32 else a for a in args) for k in range(4)]
    expected = [plain(*t) for t in tuples]
    got = list(fast.stream(iter(tuples), in_flight=2))
    assert len(got) == len(expected)
    for a, b in zip(got, expected):
        same(a, b)


@each
def test_profiled_and_with_every_value_returned(name, f, args):
    expected = mj.tree_leaves(wrap(f)(*args))
    outs, info = wrap(f, profiling=True)(*args)
    same(outs, expected)
    assert info
    outs, _ = JaxprInterpreter(mj.make_jaxpr(f)(*args), reuse_buffers=False).run(*args, return_all=True)
    same(outs, expected)


@each
def test_one_result_at_a_time(name, f, args):
    #results that nobody reads
    whole = mj.tree_leaves(wrap(f)(*args))
    for k in range(len(whole)):
        same(wrap(lambda *a: mj.tree_leaves(f(*a))[k])(*args), [whole[k]])


def test_the_same_array_in_several_places():
    x, k = normal(1, 2, 300, 40), normal(2, 3, 40)
    same(wrap(lambda x, k: nn.causal_conv(x, k, k[0], x[:, :2]))(x, k), wrap(nn.causal_conv)(x, k, k[0].copy(), x[:, :2].copy()))
    #x, widths and gate of a scan are one array, both maps another
    x, m, a = np.abs(normal(3, 2, 300, 40)) * f32(0.1), normal(4, 2, 300, 7), -np.abs(normal(5, 40, 7))
    same(wrap(lambda x, m, a: nn.selective_scan(x, x, a, m, m, gate=x))(x, m, a), wrap(lambda *v: nn.selective_scan(*v[:5], gate=v[5]))(x, x.copy(), a, m, m.copy(), x.copy()))

    def gradients(x, w, a, b, c, z, g, l):
        _, pullback = mj.vjp(lambda x, w, b, c, z: nn.selective_scan(x, w, a, b, c, gate=z), x, w, b, c, z)
        return pullback((g, l))
    g, l = normal(6, 2, 300, 40), normal(7, 2, 40, 7)
    same(wrap(lambda x, m, a, g, l: gradients(x, x, a, m, m, x, g, l))(x, m, a, g, l), wrap(gradients)(x, x.copy(), a, m, m.copy(), x.copy(), g, l))
    #the rows and the weights of a product are one array
    w, t = normal(8, 50, 50, scale=0.2), np.arange(50, dtype=np.int32)
    for transposed in (False, True):
        f = lambda x, w, t: mj.vjp(lambda x, w: nn.linear_log_probs(x, w, t, transposed), x, w)[1]((x[0], x[1]))
        same(wrap(lambda w, t: f(w, w, t))(w, t), wrap(f)(w, w.copy(), t))


@pytest.mark.parametrize('fuse', [True, False], ids=['fused', 'unfused'])
def test_operands_and_results_of_other_operations(fuse):
    '''Slices at odd offsets, transposes, broadcasts and elementwise results go in, slices of the results come out.'''
    wide, row = normal(1, 7, 90, 43), normal(2, 43)

    def conv(wide, row):
        x = jnp.transpose(wide, (1, 0, 2))[1:, :, 1:38] * np.float32(2)
        y, last = nn.causal_conv(x, jnp.broadcast_to(row[:37], (3, 37)), row[5:42], x[:, 2:4], np.arange(89, dtype=np.int32) % 9, 'silu')
        return y[3:, 1], jnp.exp(last[2])
    x = np.ascontiguousarray(wide.transpose(1, 0, 2)[1:, :, 1:38]) * f32(2)
    y, last = wrap(lambda *v: nn.causal_conv(*v, 'silu'))(x, np.ascontiguousarray(np.broadcast_to(row[:37], (3, 37))), row[5:42].copy(), x[:, 2:4].copy(), np.arange(89, dtype=np.int32) % 9)
    got = wrap(conv, fuse=fuse)(wide, row)
    same(got[0], y[3:, 1])
    close(got[1], np.exp(last[2].astype(np.float64)), 8 * U * np.exp(last[2].astype(np.float64)))

    arrays, _, _ = scan_inputs(3, 50, 21, 6, ('gate',), False)
    joined = np.concatenate([arrays[k] for k in ('x', 'delta', 'gate', 'b', 'c')], axis=2)

    def scan(joined, a):
        x, delta, gate, b, c = joined[:, :, :21], joined[:, :, 21:42], joined[:, :, 42:63], joined[:, :, 63:69], joined[:, :, 69:]
        y, last = nn.selective_scan(x, delta, jnp.transpose(a), b, c, gate=gate)
        return y[:, 7:9, 3:], last[1:]
    y, last = wrap(lambda *v: nn.selective_scan(*v[:5], gate=v[5]))(*(arrays[k] for k in ('x', 'delta', 'a', 'b', 'c', 'gate')))
    same(wrap(scan, fuse=fuse)(joined, np.ascontiguousarray(arrays['a'].T)), (y[:, 7:9, 3:], last[1:]))

    table = normal(3, 31, 450)
    ids = np.array([[4, 2, 89], [0, -1, 90]], np.int32)

    def probs(table, ids):
        x = jnp.reshape(table[3:9, 7:57], (3, 2, 50))
        lp, ls = nn.linear_log_probs(x, jnp.transpose(table[10:, 25:75] * np.float32(0.5)), jnp.transpose(ids) - np.int32(1))
        return lp[1:], ls[:, 1]
    lp, ls = wrap(nn.linear_log_probs)(table[3:9, 7:57].reshape(3, 2, 50).copy(), np.ascontiguousarray(table[10:, 25:75].T) * f32(0.5), np.ascontiguousarray(ids.T) - 1)
    same(wrap(probs, fuse=fuse)(table, ids), (lp[1:], ls[:, 1]))
    m = normal(4, 70, 2, 31)
    same(wrap(lambda m: nn.orthogonalize(jnp.transpose(m, (1, 0, 2))[1, 3:, 1:], 2)[5:], fuse=fuse)(m), wrap(lambda m: nn.orthogonalize(m, 2))(m[3:, 1, 1:].copy())[5:])


def test_arrays_of_the_host_in_any_form():
    x, k = np.asfortranarray(normal(1, 3, 20, 12).astype(np.float64)), normal(2, 12, 4).T
    same(wrap(nn.causal_conv)(x, k), wrap(nn.causal_conv)(np.ascontiguousarray(x, f32), np.ascontiguousarray(k)))
    x, w, t = normal(3, 9, 80).T, normal(4, 50, 18)[:, ::2].T.astype(np.float64), np.arange(80, dtype=np.int64) % 50
    same(wrap(nn.linear_log_probs)(x, w, t), wrap(nn.linear_log_probs)(np.ascontiguousarray(x), np.ascontiguousarray(w, f32), t.astype(np.int32)))
    m = normal(5, 40, 60)[::-1, ::2]
    same(wrap(nn.orthogonalize)(m), wrap(nn.orthogonalize)(m.copy()))


# ------------------------------------------------------------------ arrays whose offsets pass 31 bits, and 32

def test_convolutions_of_more_than_four_gigabytes():
    '''x[b, t, c] = a[t] r[c]: of its results the last times of the last sequence.'''
    t, c = 850001, 1300
    a, r, k = normal(1, t), normal(2, c), normal(3, 4, c)

    def f(a, r, k):
        x = jnp.reshape(a, (1, t, 1)) * jnp.reshape(r, (1, 1, c))
        (y, last), pullback = mj.vjp(lambda x, k: nn.causal_conv(x, k), x, k)
        dx, dk = pullback((x, jnp.zeros((1, 3, c), np.float32)))
        return y[0, t - 5:], last[0], dx[0, t - 5:], dk
    y, last, dx, dk = wrap(f)(a, r, k)
    a64, r64, k64 = a.astype(np.float64), r.astype(np.float64), k.astype(np.float64)
    rows = (a[-8:, None] * r[None]).astype(f32).astype(np.float64)
    assert np.array_equal(last, rows[-3:].astype(f32))
    size = np.abs(rows).max() * np.abs(k64).sum(0)
    close(y, sum(k64[i] * rows[i:i + 5] for i in range(4)), 6 * U * size)
    behind = np.concatenate([rows[3:], np.zeros((3, c))])
    close(dx, sum(k64[3 - j] * behind[j:j + 5] for j in range(4)), 6 * U * size)
    #dk[i] = r^2 sum a[t] a[t - 3 + i]; x is rounded twice, sums of n terms in a lane (up to 8 times as many steps as tiles of time take turns), a block and over blocks in turn
    for i in range(4):
        expected = r64 ** 2 * (a64[3 - i:] * a64[:t - 3 + i]).sum()
        close(dk[i], expected, 4000 * U * r64 ** 2 * np.abs(a64[3 - i:] * a64[:t - 3 + i]).sum())


def test_scans_of_more_than_four_gigabytes():
    '''The same operands at every time: the last times of the last sequence, in which a state has long come to where it stays.'''
    b, t, c, n = 2, 450001, 1300, 4
    a, r = -(0.5 + np.random.default_rng(1).random((c, n))).astype(f32), normal(2, c)

    def f(a, r):
        x = jnp.broadcast_to(jnp.reshape(r, (1, 1, c)), (b, t, c))
        one = jnp.ones((b, t, n), np.float32)
        y, last = nn.selective_scan(x, jnp.full((b, t, c), np.float32(0.25)), a, one, one)
        return y[b - 1, t - 5:], last[b - 1]
    y, last = wrap(f)(a, r)
    factor = np.exp(0.25 * a.astype(np.float64))
    h = 0.25 * r.astype(np.float64)[:, None] / (1 - factor)
    #(a factor is off by some 4 u, the state by 4 u / (1 - factor) of itself and one rounding per step, of which 1 / (1 - factor) stay)
    bound = 8 * U * np.abs(h) / (1 - factor)
    close(last, h, bound)
    close(y, np.broadcast_to(h.sum(1), (5, c)), (bound + 4 * U * np.abs(h)).sum(1))


def test_gradient_of_scans_of_two_gigabytes():
    '''States that forget at once (a = -200): the gradient of a step is its own.'''
    t, c = 430001, 1300
    x, g = normal(1, t), normal(2, c)

    def f(x, g):
        xs = jnp.broadcast_to(jnp.reshape(x, (1, t, 1)), (1, t, c))
        gs = jnp.broadcast_to(jnp.reshape(g, (1, 1, c)), (1, t, c))
        one, w = jnp.ones((1, t, 1), np.float32), jnp.full((1, t, c), np.float32(1))
        (y, _), pullback = mj.vjp(lambda x, b: nn.selective_scan(x, w, jnp.full((c, 1), np.float32(-200)), b, one), xs, one)
        dx, db = pullback((gs, jnp.zeros((1, c, 1), np.float32)))
        return y[0, t - 5:], dx[0, t - 5:], db[0, t - 5:]
    y, dx, db = wrap(f)(x, g)
    assert np.array_equal(y, np.broadcast_to(x[-5:, None], (5, c))) and np.array_equal(dx, np.broadcast_to(g, (5, c)))
    close(db[:, 0], x[-5:].astype(np.float64) * g.astype(np.float64).sum(), 24 * U * np.abs(x[-5:]) * np.abs(g).sum())


@pytest.mark.parametrize('rows,transposed', [(3, False), (3, True), (70, False), (70, True)])
def test_log_probs_from_weights_of_more_than_four_gigabytes(rows, transposed):
    '''W[h, v] = p[h] q[v]: scores are (x . p) q[v]. Of dx everything, of dW the last columns.'''
    h, v = 4097, 280003
    p, q, x = normal(1, h, scale=h ** -0.5), normal(2, v), normal(3, rows, h)
    t = (np.arange(rows) * 12345 % v).astype(np.int32)
    t[0], t[1] = v - 1, -1

    def f(p, q, x, t):
        w = jnp.reshape(q, (v, 1)) * jnp.reshape(p, (1, h)) if transposed else jnp.reshape(p, (h, 1)) * jnp.reshape(q, (1, v))
        (lp, ls), pullback = mj.vjp(lambda x, w: nn.linear_log_probs(x, w, t, transposed), x, w)
        dx, dw = pullback((lp * np.float32(0) + np.float32(1), lp * np.float32(0)))
        return lp, ls, dx, dw[v - 3:] if transposed else jnp.transpose(dw[:, v - 3:])
    lp, ls, dx, dw = wrap(f)(p, q, x, t)
    x64, p64, q64 = x.astype(np.float64), p.astype(np.float64), q.astype(np.float64)
    given = t >= 0
    s = x64 @ p64
    scores = s[:, None] * q64
    peak = scores.max(1)
    prob = np.exp(scores - peak[:, None])
    total = prob.sum(1)
    prob /= total[:, None]
    at = np.where(given, t, 0)
    expected = scores[np.arange(rows), at] - peak - np.log(total)
    #scores: weights are rounded once, a sum of 4097 terms is off by 512 + 24 roundings at most (most of the bound)
    e_s = 540 * U * (np.abs(x64) @ np.abs(p64)) * np.abs(q64).max()
    close(lp, np.where(given, expected, 0), np.where(given, 2 * e_s + 300 * U + 8 * U * np.abs(peak), 0))
    close(ls, np.where(given, peak + np.log(total), 0), np.where(given, e_s + 300 * U + 8 * U * np.abs(peak), 0))
    e_p = 3 * e_s + 600 * U                                                                 #of a probability, relative
    dq = q64[at] - prob @ q64
    close(dx, np.where(given[:, None], dq[:, None] * p64, 0), np.where(given[:, None], (e_p * (prob @ np.abs(q64)) + 36000 * U * (prob @ np.abs(q64)) + 8 * U * np.abs(q64[at]))[:, None] * np.abs(p64) + 1e-30, 0))
    ds = np.where(given[:, None], -prob[:, -3:], 0)
    ds[0, 2] += 1
    close(dw, ds.T @ x64, (np.abs(ds) * (e_p + 40 * U)[:, None]).T @ np.abs(x64) + 1e-30)


def test_orthogonalising_more_than_four_gigabytes():
    '''x = r s^T, of rank one: x / |x| again (its one singular value, 1, stays). Of the results the last rows.'''
    rows, columns = 1100, 1000003
    r, s = normal(1, rows), normal(2, columns)
    r64, s64 = r.astype(np.float64), s.astype(np.float64)
    norm = np.sqrt((r64 ** 2).sum() * (s64 ** 2).sum())
    for tall in (False, True):
        def f(r, s):
            x = jnp.reshape(s, (columns, 1)) * jnp.reshape(r, (1, rows)) if tall else jnp.reshape(r, (rows, 1)) * jnp.reshape(s, (1, columns))
            return nn.orthogonalize(x, 1, (1.5, -0.5, 0.0))[-2:]
        expected = (s64[-2:, None] * r64 if tall else r64[-2:, None] * s64) / norm
        #the norm's sum of squares is off by some 1000 u at most, products by far less
        close(wrap(f)(r, s), expected, 2.0 ** -11 * np.abs(expected).max())
