'''Operators of a recurrent token model that is trained and served - its mixing layer, its loss and its update -, over the sizes in
which they are used:

* `causal_conv`: a short causal convolution along time, channel by channel, `nn.causal_conv(x, kernel, bias, state, lengths,
  activation)`;
* `selective_scan`: a state space whose step widths and input and output maps come from the data, `nn.selective_scan(x, delta, a,
  b, c, d, gate, state, lengths, delta_bias, softplus)`;
* `linear_log_probs`: log probabilities of given tokens under the softmax of a product with the vocabulary's weights, in pieces of
  the vocabulary, without keeping the scores, `nn.linear_log_probs(x, weights, tokens, transposed)`;
* `orthogonalize`: a matrix of gradients with its singular values brought to about 1 by products of matrices,
  `nn.orthogonalize(x, steps)`.

A case is a program of one operator: its forward pass (`way='forward'`), or its forward and backward pass for given cotangents
(`way='train'`: `mj.vjp`). The framework's programs work on arguments that lie in HBM and leave their results there
(`JaxprInterpreter.upload_inputs` / `.replay`), as a program does whose data stay on the device. The plain forms compute the
same from elementary torch operations.
'''
import ctypes

import numpy as np
import torch

own = False

DEVICE = 'cuda'
#the polynomial of a step, a s + b s^3 + c s^5 of the singular values s
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
ORTHOGONAL_EPS = 1e-7


# ------------------------------------------------------------------ the cases

def listed():
    return [
        #one token of each of 64 sequences that are decoded together: the smallest call, latency only
        dict(name='conv_token', op='causal_conv', way='forward', batch=64, time=1, channels=2048, width=4, state=True, ragged=False, activation='silu'),
        #a training step over a padded batch
        dict(name='conv_train', op='causal_conv', way='train', batch=8, time=2048, channels=2048, width=4, state=False, ragged=True, activation='silu'),
        #odd sizes, without an activation, going on from a state
        dict(name='conv_ragged', op='causal_conv', way='train', batch=3, time=1021, channels=333, width=3, state=True, ragged=True, activation='none'),
        #one token of each of 64 sequences: the states are read and written, little else
        dict(name='scan_token', op='selective_scan', way='forward', batch=64, time=1, channels=2048, states=16, state=True, ragged=False, gated=True, softplus=True),
        #a long prompt read at once, one sequence
        dict(name='scan_prompt', op='selective_scan', way='forward', batch=1, time=16384, channels=2048, states=16, state=True, ragged=False, gated=True, softplus=True),
        #a training step over a padded batch
        dict(name='scan_train', op='selective_scan', way='train', batch=4, time=2048, channels=2048, states=16, state=False, ragged=True, gated=True, softplus=True),
        #odd sizes, step widths as they are, no gate
        dict(name='scan_ragged', op='selective_scan', way='train', batch=3, time=1021, channels=333, states=7, state=True, ragged=True, gated=False, softplus=False),
        #eight served sequences: the probability of the token that each was given
        dict(name='loss_decode', op='linear_log_probs', way='forward', rows=8, hidden=1024, vocabulary=32000, padded=0, tied=False),
        #a training step's loss, some positions padded
        dict(name='loss_train', op='linear_log_probs', way='train', rows=4096, hidden=1024, vocabulary=32000, padded=256, tied=False),
        #fewer rows, odd sizes, the weights of the embedding used again (a row per token)
        dict(name='loss_tied', op='linear_log_probs', way='train', rows=321, hidden=500, vocabulary=50001, padded=7, tied=True),
        #the layers of a small model, stacked
        dict(name='orthogonal_layers', op='orthogonalize', way='forward', matrices=12, rows=512, columns=512, steps=5),
        #one large layer
        dict(name='orthogonal_large', op='orthogonalize', way='forward', matrices=1, rows=4096, columns=4096, steps=5),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def _width(rng, low, high):
    '''A number of channels: mostly a multiple of 8, at times any number.'''
    n = _log_int(rng, low, high)
    return n if rng.random() < 0.3 else max(low, n // 8 * 8)


def draw(rng):
    op = rng.choice(('causal_conv', 'selective_scan', 'linear_log_probs', 'orthogonalize'))
    case = dict(op=op, way='forward' if op == 'orthogonalize' else rng.choice(('forward', 'train')))
    if op in ('causal_conv', 'selective_scan'):
        channels, states = _width(rng, 8, 4096), 1
        if op == 'selective_scan':
            states = rng.choice((1, 4, 8, 16, 16, 16, 24, 32, 64))
        room = 33e6 if op == 'causal_conv' else (5e8 if case['way'] == 'forward' else 2.6e8)
        time = rng.choice((1, _log_int(rng, 2, 16384), _log_int(rng, 2, 16384)))
        time = max(1, min(time, int(room // (channels * states))))
        batch = _log_int(rng, 1, max(1, min(64, int(room // (time * channels * states)))))
        case.update(batch=batch, time=time, channels=channels, state=rng.random() < 0.5, ragged=rng.random() < 0.5)
        if op == 'causal_conv':
            case.update(width=rng.choice((2, 3, 4, 4, 4, 8)), activation=rng.choice(('none', 'silu')))
        else:
            case.update(states=states, gated=rng.random() < 0.6, softplus=rng.random() < 0.6)
    elif op == 'linear_log_probs':
        vocabulary, hidden = _log_int(rng, 100, 131072), _width(rng, 32, 4096)
        most = max(1, min(16384, int(1.3e11 // (vocabulary * hidden)), int(1.3e8 // vocabulary)))
        rows = _log_int(rng, 1, most)
        case.update(rows=rows, hidden=hidden, vocabulary=vocabulary, padded=rng.choice((0, rows // 8)), tied=rng.random() < 0.4)
    else:
        rows, columns = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
        small = min(rows, columns)
        most = max(1, min(32, int(6.8e10 // (small * small * max(rows, columns)))))
        case.update(matrices=_log_int(rng, 1, most), rows=rows, columns=columns, steps=rng.choice((1, 3, 5, 5)))
    return case


# ------------------------------------------------------------------ inputs

def _lengths(case, turn=0):
    '''Lengths between half and all of the padded time, spread evenly; the sequence they start with differs by seed.'''
    b, t = case['batch'], case['time']
    return [t - ((i + turn) % b) * t // (2 * b) for i in range(b)]


def _inputs(case, seed):
    '''{name: tensor on the GPU}, from the seed alone.'''
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).mul_(scale).add_(shift)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEVICE, dtype=torch.float32)

    def integers(n, *shape):
        return torch.randint(0, n, shape, generator=g, device=DEVICE, dtype=torch.int32)

    train = case['way'] == 'train'
    if case['op'] == 'orthogonalize':
        #what a momentum of gradients looks like: a few directions that stand out, and noise
        m, r, c = case['matrices'], case['rows'], case['columns']
        few = min(8, r, c)
        x = normal(m, r, c, scale=1e-3)
        for i in range(few):
            x += normal(m, r, 1) * normal(m, 1, c, scale=4e-3 * 0.7 ** i)
        return dict(x=x)
    if case['op'] == 'linear_log_probs':
        rows, h, v = case['rows'], case['hidden'], case['vocabulary']
        weights = normal(v, h, scale=2.0 * h ** -0.5) if case['tied'] else normal(h, v, scale=2.0 * h ** -0.5)
        tokens = integers(v, rows)
        if case['padded']:
            tokens[torch.randperm(rows, generator=g, device=DEVICE)[:case['padded']]] = -1
        found = dict(x=normal(rows, h), weights=weights, tokens=tokens)
        if train:
            #a mean over the rows, and a small pull on the log of the sum
            found['g_log_probs'] = normal(rows, scale=0.2 / rows, shift=-1.0 / rows)
            found['g_log_sums'] = normal(rows, scale=0.01 / rows)
        return found
    b, t, c = case['batch'], case['time'], case['channels']
    found = dict(x=normal(b, t, c))
    if case['op'] == 'causal_conv':
        k = case['width']
        found.update(kernel=normal(k, c, scale=k ** -0.5), bias=normal(c, scale=0.1))
        if case['state']:
            found['state'] = normal(b, k - 1, c)
    else:
        n = case['states']
        if case['softplus']:
            #step widths between 0.001 and 0.1 where the projection adds nothing
            found['delta'] = normal(b, t, c, scale=0.5)
            found['delta_bias'] = torch.log(torch.expm1(10.0 ** (-3.0 + 2.0 * uniform(c))))
        else:
            found['delta'] = 10.0 ** (-3.0 + 2.0 * uniform(b, t, c))
        found['a'] = -(0.5 + uniform(c, n)) * torch.arange(1, n + 1, device=DEVICE, dtype=torch.float32)
        found.update(b=normal(b, t, n), c=normal(b, t, n), d=0.5 + uniform(c))
        if case['gated']:
            found['gate'] = normal(b, t, c)
        if case['state']:
            found['state'] = normal(b, c, n, scale=0.3)
    if case['ragged']:
        found['lengths'] = torch.tensor(_lengths(case, int(integers(b, 1).item())), dtype=torch.int32, device=DEVICE)
    if train:
        found['g'] = normal(b, t, c)
        found['g_last'] = normal(b, case['width'] - 1, c) if case['op'] == 'causal_conv' else normal(b, c, case['states'])
    return found


# ------------------------------------------------------------------ the framework's programs

class _InHBM:
    '''A result array of a recorded program where it lies in HBM.'''
    def __init__(self, buffer):
        kind = '<f4' if buffer.dtype == np.float32 else '<i4'
        self.owner = buffer
        self.__cuda_array_interface__ = dict(shape=buffer.shape, typestr=kind, data=(buffer.tensor.device_ptr(), False), version=2)


#the operands with a gradient, in the order in which the results hold them
_WITH_GRADIENTS = {'causal_conv': ('x', 'kernel', 'bias', 'state'),
                   'selective_scan': ('x', 'delta', 'a', 'b', 'c', 'd', 'gate', 'state', 'delta_bias'),
                   'linear_log_probs': ('x', 'weights')}
_COTANGENTS = {'causal_conv': ('g', 'g_last'), 'selective_scan': ('g', 'g_last'), 'linear_log_probs': ('g_log_probs', 'g_log_sums')}


def _program(case, names):
    '''A function of the arrays `names` for the framework to trace.'''
    from vkjax_amd import minijax as mj
    nn = mj.nn

    def forward(a):
        if case['op'] == 'orthogonalize':
            return nn.orthogonalize(a['x'], steps=case['steps'], coefficients=COEFFICIENTS, eps=ORTHOGONAL_EPS)
        if case['op'] == 'linear_log_probs':
            return nn.linear_log_probs(a['x'], a['weights'], a['tokens'], transposed=case['tied'])
        if case['op'] == 'causal_conv':
            return nn.causal_conv(a['x'], a['kernel'], a['bias'], state=a.get('state'), lengths=a.get('lengths'),
                                  activation=None if case['activation'] == 'none' else case['activation'])
        return nn.selective_scan(a['x'], a['delta'], a['a'], a['b'], a['c'], d=a['d'], gate=a.get('gate'), state=a.get('state'),
                                 lengths=a.get('lengths'), delta_bias=a.get('delta_bias'), softplus=case['softplus'])

    def run_forward(*arrays):
        return forward(dict(zip(names, arrays)))

    def run_train(*arrays):
        a = dict(zip(names, arrays))
        wrt = [n for n in _WITH_GRADIENTS[case['op']] if n in a]
        outs, pullback = mj.vjp(lambda *values: forward(dict(a, **dict(zip(wrt, values)))), *[a[n] for n in wrt])
        return tuple(outs) + tuple(pullback(tuple(a[n] for n in _COTANGENTS[case['op']])))
    return run_forward if case['way'] == 'forward' else run_train


def _recorded(case, arrays):
    '''The framework's program with its arguments in HBM, and its results there.'''
    from vkjax_amd import minijax as mj
    from vkjax_amd.jaxpr_interpreter import JaxprInterpreter
    host = [a.cpu().numpy() for a in arrays.values()]
    program = JaxprInterpreter(mj.make_jaxpr(_program(case, list(arrays)))(*host))
    program.upload_inputs(*host)
    #a kernel is looked for in one code object after the other; the status of the last one that does not hold it would be
    #reported by torch's next call in its own name
    ctypes.CDLL('libamdhip64.so.7').hipGetLastError()
    return dict(program=program, outputs=[torch.as_tensor(_InHBM(b), device=DEVICE) for b in program.output_buffers])


def prepare(case, seed):
    arrays = _inputs(case, seed)
    if own:
        return _recorded(case, arrays)
    return dict(case=case, arrays=arrays)


def run(state):
    if own:
        state['program'].replay(1)
        return state['outputs']
    case = state['case']
    plain = {'causal_conv': _plain_conv, 'selective_scan': _plain_scan, 'linear_log_probs': _plain_loss, 'orthogonalize': _plain_orthogonal}
    return plain[case['op']](case, **state['arrays'])


# ------------------------------------------------------------------ the plain forms

def _inside(x, lengths):
    '''Where a sequence has not ended, [batch, time, 1], or None.'''
    return None if lengths is None else torch.arange(x.shape[1], device=x.device)[None, :, None] < lengths[:, None, None]


def _kept(v, inside):
    return v if inside is None else torch.where(inside, v, torch.zeros_like(v))


def _plain_conv(case, x, kernel, bias, state=None, lengths=None, g=None, g_last=None):
    (b, t, c), k = x.shape, kernel.shape[0]
    inside = _inside(x, lengths)
    before = x.new_zeros(b, k - 1, c) if state is None else state
    whole = torch.cat([before, _kept(x, inside)], dim=1)
    z = bias.expand(b, t, c)
    for i in range(k):
        z = z + whole[:, i:i + t] * kernel[i]
    gate = 1.0 / (1.0 + torch.exp(-z)) if case['activation'] == 'silu' else None
    y = _kept(z if gate is None else z * gate, inside)
    ends = torch.full((b,), t, device=x.device) if lengths is None else lengths.long()
    rows = (ends[:, None] + torch.arange(k - 1, device=x.device)[None])[:, :, None].expand(b, k - 1, c)
    outs = [y, whole.gather(1, rows)]
    if g is None:
        return outs
    d = _kept(g if gate is None else g * gate * (1.0 + z * (1.0 - gate)), inside)
    dwhole = torch.zeros_like(whole)
    for i in range(k):
        dwhole[:, i:i + t] += d * kernel[i]
    dwhole.scatter_add_(1, rows, g_last)
    dkernel = torch.stack([(d * whole[:, i:i + t]).sum(dim=(0, 1)) for i in range(k)])
    return outs + [_kept(dwhole[:, k - 1:], inside), dkernel, d.sum(dim=(0, 1))] + ([dwhole[:, :k - 1]] if state is not None else [])


def _scan(a, h):
    '''h[t] = a[t] h[t-1] + h[t] along axis 1 from 0, by doubling, in place (a is used up).'''
    step = 1
    while step < h.shape[1]:
        h[:, step:] += a[:, step:] * h[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return h


def _plain_scan(case, x, delta, a, b, c, d, gate=None, state=None, lengths=None, delta_bias=None, g=None, g_last=None):
    inside = _inside(x, lengths)
    v = delta if delta_bias is None else delta + delta_bias
    width = torch.where(v > 0, v, torch.zeros_like(v)) + torch.log1p(torch.exp(-v.abs())) if case['softplus'] else v
    width, u = _kept(width, inside), _kept(x, inside)
    factor = torch.exp(width[..., None] * a)
    h = (width * u)[..., None] * b[:, :, None, :]
    if state is not None:
        h[:, 0] += factor[:, 0] * state
    h = _scan(factor.clone() if g is not None else factor, h)
    last = h[:, -1].clone()
    seen = (h * c[:, :, None, :]).sum(dim=3) + d * u
    open_ = None if gate is None else 1.0 / (1.0 + torch.exp(-gate))
    y = _kept(seen if gate is None else seen * gate * open_, inside)
    if g is None:
        return [y, last]
    g = _kept(g, inside)
    dgate = None
    if gate is not None:
        dgate = g * seen * open_ * (1.0 + gate * (1.0 - open_))
        g = g * gate * open_
    dc = _kept((h * g[..., None]).sum(dim=2), inside)
    #the adjoint runs the other way: l[t] = g[t] c[t] + factor[t+1] l[t+1]
    l = g[..., None] * c[:, :, None, :]
    l[:, -1] += g_last
    back = torch.cat([factor[:, 1:], torch.ones_like(factor[:, :1])], dim=1).flip(1)
    l = _scan(back, l.flip(1)).flip(1)
    del back
    dstate = factor[:, 0] * l[:, 0]
    first = torch.zeros_like(h[:, :1]) if state is None else state[:, None]
    e = factor.mul_(l).mul_(torch.cat([first, h[:, :-1]], dim=1))          #the cotangent of width * a
    del h
    da = (e * width[..., None]).sum(dim=(0, 1))
    through = (l * b[:, :, None, :]).sum(dim=3)
    dwidth = _kept((e * a).sum(dim=3) + through * u, inside)
    dx = _kept(through * width + d * g, inside)
    db = _kept((l * (width * u)[..., None]).sum(dim=2), inside)
    ddelta = dwidth / (1.0 + torch.exp(-v)) if case['softplus'] else dwidth
    found = [dx, ddelta, da, db, dc, (g * u).sum(dim=(0, 1))]
    found += [dgate] if gate is not None else []
    found += [dstate] if state is not None else []
    found += [ddelta.sum(dim=(0, 1))] if delta_bias is not None else []
    return [y, last] + found


def _plain_loss(case, x, weights, tokens, g_log_probs=None, g_log_sums=None):
    w = weights.t() if case['tied'] else weights
    v = w.shape[1]
    given = (tokens >= 0) & (tokens < v)
    at = torch.where(given, tokens, torch.zeros_like(tokens)).long()[:, None]
    scores = x @ w
    best = scores.max(dim=1, keepdim=True).values
    e = torch.exp(scores - best)
    total = e.sum(dim=1, keepdim=True)
    log_sums = best + torch.log(total)
    zero = torch.zeros((), device=x.device)
    outs = [torch.where(given, (scores.gather(1, at) - log_sums)[:, 0], zero), torch.where(given, log_sums[:, 0], zero)]
    if g_log_probs is None:
        return outs
    of_token, of_sum = torch.where(given, g_log_probs, zero), torch.where(given, g_log_sums - g_log_probs, zero)
    d = (e / total) * of_sum[:, None]
    d.scatter_add_(1, at, of_token[:, None])
    dw = d.t() @ x if case['tied'] else x.t() @ d
    return outs + [d @ w.t(), dw]


def _plain_orthogonal(case, x):
    a, b, c = COEFFICIENTS
    tall = x.shape[1] > x.shape[2]
    m = x.transpose(1, 2) if tall else x
    m = m / ((m * m).sum(dim=(1, 2), keepdim=True).sqrt() + ORTHOGONAL_EPS)
    for _ in range(case['steps']):
        square = torch.bmm(m, m.transpose(1, 2).contiguous())
        m = a * m + torch.bmm(b * square + c * torch.bmm(square, square), m)
    return [m.transpose(1, 2).contiguous() if tall else m]


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    a = {k: v.double() if v.dtype == torch.float32 else v for k, v in _inputs(case, seed).items()}
    found = {'causal_conv': _exact_conv, 'selective_scan': _exact_scan, 'linear_log_probs': _exact_loss, 'orthogonalize': _exact_orthogonal}
    return found[case['op']](case, **a)


def _exact_conv(case, x, kernel, bias, state=None, lengths=None, g=None, g_last=None):
    batch, time, channels = x.shape
    k = kernel.shape[0]
    ends = [time] * batch if lengths is None else lengths.tolist()
    ys, lasts, dxs, dstates = [], [], [], []
    dkernel, dbias = torch.zeros_like(kernel), torch.zeros_like(bias)
    for i, n in enumerate(ends):
        first = torch.zeros(k - 1, channels, dtype=x.dtype, device=x.device) if state is None else state[i]
        rows = torch.cat([first, x[i, :n]])
        windows = rows.unfold(0, k, 1)                                   #[n, channels, k]
        z = torch.einsum('tck,kc->tc', windows, kernel) + bias
        s = torch.sigmoid(z)
        act, slope = (z * s, s + z * s * (1 - s)) if case['activation'] == 'silu' else (z, torch.ones_like(z))
        fill = torch.zeros(time - n, channels, dtype=x.dtype, device=x.device)
        ys.append(torch.cat([act, fill]))
        lasts.append(rows[n:])
        if g is None:
            continue
        d = g[i, :n] * slope
        dbias += d.sum(0)
        dkernel += torch.einsum('tck,tc->kc', windows, d)
        padded = torch.cat([torch.zeros_like(first), d, torch.zeros_like(first)]).unfold(0, k, 1)    #[n + k - 1, channels, k]
        drows = torch.einsum('tck,kc->tc', padded, kernel.flip(0))
        drows[n:] += g_last[i]
        dstates.append(drows[:k - 1])
        dxs.append(torch.cat([drows[k - 1:], fill]))
    outs = [torch.stack(ys), torch.stack(lasts)]
    if g is None:
        return outs
    return outs + [torch.stack(dxs), dkernel, dbias] + ([torch.stack(dstates)] if state is not None else [])


def _exact_scan(case, x, delta, a, b, c, d, gate=None, state=None, lengths=None, delta_bias=None, g=None, g_last=None):
    batch, time, channels = x.shape
    ends = torch.full((batch,), time, device=x.device) if lengths is None else lengths.long()
    pre = delta if delta_bias is None else delta + delta_bias
    dt = torch.nn.functional.softplus(pre, threshold=50.0) if case['softplus'] else pre.clone()
    live = (torch.arange(time, device=x.device)[None] < ends[:, None])
    dt[~live] = 0.0
    u = x.clone()
    u[~live] = 0.0
    now = torch.zeros(batch, channels, a.shape[1], dtype=x.dtype, device=x.device) if state is None else state.clone()
    out = torch.empty_like(x)
    states = None if g is None else torch.empty(time + 1, *now.shape, dtype=x.dtype, device=x.device)
    for t in range(time):
        if states is not None:
            states[t] = now
        now = torch.exp(dt[:, t, :, None] * a) * now + torch.einsum('bc,bn->bcn', dt[:, t] * u[:, t], b[:, t])
        out[:, t] = torch.einsum('bcn,bn->bc', now, c[:, t]) + d * u[:, t]
    shut = torch.nn.functional.silu(gate) if gate is not None else torch.ones_like(x)
    y = out * shut * live[:, :, None]
    if g is None:
        return [y, now]
    states[time] = now
    gy = g * live[:, :, None]
    dgate = None
    if gate is not None:
        s = torch.sigmoid(gate)
        dgate, gy = gy * out * (s + gate * s * (1 - s)), gy * shut
    dx, ddt = torch.empty_like(x), torch.empty_like(x)
    db, dc, da, l = torch.empty_like(b), torch.empty_like(c), torch.zeros_like(a), g_last.clone()
    for t in range(time - 1, -1, -1):
        f = torch.exp(dt[:, t, :, None] * a)
        l = l + torch.einsum('bc,bn->bcn', gy[:, t], c[:, t])
        dc[:, t] = torch.einsum('bcn,bc->bn', states[t + 1], gy[:, t])
        lb = torch.einsum('bcn,bn->bc', l, b[:, t])
        db[:, t] = torch.einsum('bcn,bc->bn', l, dt[:, t] * u[:, t])
        e = l * f * states[t]
        da += torch.einsum('bcn,bc->cn', e, dt[:, t])
        ddt[:, t] = torch.einsum('bcn,cn->bc', e, a) + lb * u[:, t]
        dx[:, t] = lb * dt[:, t] + d * gy[:, t]
        l = l * f
    for v in (dx, ddt, db, dc):
        v[~live] = 0.0
    ddelta = ddt * torch.sigmoid(pre) if case['softplus'] else ddt
    found = [dx, ddelta, da, db, dc, (gy * u).sum(dim=(0, 1))]
    found += [dgate] if gate is not None else []
    found += [l] if state is not None else []
    found += [ddelta.sum(dim=(0, 1))] if delta_bias is not None else []
    return [y, now] + found


def _exact_loss(case, x, weights, tokens, g_log_probs=None, g_log_sums=None):
    w = weights.mT if case['tied'] else weights
    rows, v = x.shape[0], w.shape[1]
    log_probs, log_sums = x.new_zeros(rows), x.new_zeros(rows)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for i in range(0, rows, 1024):                                       #some rows at a time: 64 bits take room
        part = torch.arange(i, min(rows, i + 1024), device=x.device)
        part = part[(tokens[part] >= 0) & (tokens[part] < v)]
        token = tokens[part].long()
        z = torch.matmul(x[part], w)
        log_sums[part] = torch.logsumexp(z, dim=1)
        log_probs[part] = z.gather(1, token[:, None])[:, 0] - log_sums[part]
        if g_log_probs is not None:
            d = torch.softmax(z, dim=1) * (g_log_sums[part] - g_log_probs[part])[:, None]
            d[torch.arange(len(part), device=x.device), token] += g_log_probs[part]
            dx[part] = torch.matmul(d, w.mT)
            dw += torch.matmul(x[part].mT, d)
    outs = [log_probs, log_sums]
    return outs if g_log_probs is None else outs + [dx, dw.mT.contiguous() if case['tied'] else dw]


def _exact_orthogonal(case, x):
    a, b, c = COEFFICIENTS
    found = []
    for m in x:
        m = m / (torch.linalg.vector_norm(m) + ORTHOGONAL_EPS)
        #a function of the singular values, taken from whichever side is smaller
        left = m.shape[0] <= m.shape[1]
        eye = torch.eye(min(m.shape), dtype=m.dtype, device=m.device)
        for _ in range(case['steps']):
            s = m @ m.mT if left else m.mT @ m
            p = a * eye + s @ (b * eye + c * s)
            m = p @ m if left else m @ p
        found.append(m)
    return [torch.stack(found)]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    train = case['way'] == 'train'
    if case['op'] == 'orthogonalize':
        m, r, c = case['matrices'], min(case['rows'], case['columns']), max(case['rows'], case['columns'])
        #(squares are symmetric: half their products)
        return dict(bytes=8 * m * r * c, flops=m * case['steps'] * (r * r * c + r * r * r + 2 * r * r * c))
    if case['op'] == 'linear_log_probs':
        rows, h, v = case['rows'], case['hidden'], case['vocabulary']
        given = rows - case['padded']
        return dict(bytes=4 * ((given * h + h * v) * (2 if train else 1) + rows * (5 if train else 3)), flops=2 * given * h * v * (3 if train else 1))
    b, t, c = case['batch'], case['time'], case['channels']
    inside = sum(_lengths(case)) if case['ragged'] else b * t
    if case['op'] == 'causal_conv':
        k = case['width']
        ends = b * (k - 1) * c * (1 + case['state'])
        small = (k + 1) * c
        if not train:
            return dict(bytes=4 * (inside * c + b * t * c + ends + small), flops=inside * c * (2 * k + (4 if case['activation'] == 'silu' else 0)))
        return dict(bytes=4 * (2 * inside * c + 2 * b * t * c + 2 * ends + 2 * small), flops=inside * c * (6 * k + (12 if case['activation'] == 'silu' else 0)))
    n = case['states']
    per_step = 2 + case['gated']                                         #x, delta, gate
    ends = b * c * n * (1 + case['state'])
    if not train:
        return dict(bytes=4 * (inside * (per_step * c + 2 * n) + b * t * c + ends + c * (n + 2)), flops=inside * c * (n * 7 + 8))
    return dict(bytes=4 * (inside * ((per_step + 1) * c + 2 * n) + b * t * ((1 + per_step) * c + 2 * n) + 2 * ends + 2 * c * (n + 2)),
                flops=inside * c * (n * 24 + 24))
