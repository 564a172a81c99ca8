'''Operators of token models and of networks that are trained with their normalisation, over the sizes in which they are used:

* `group_norm`: group norm of channels-last activations with the activation behind it,
  `nn.group_norm(x, scale, shift, groups, eps, activation)`;
* `token_log_probs`: log probabilities of given tokens (or classes) with the entropy of each row's distribution and its most
  likely alternatives, `nn.token_log_probs(logits, tokens, top)`;
* `recurrence`: h[t] = a[t] h[t-1] + (1 - a[t]) x[t] with a = sigmoid(gate), `nn.gated_recurrence(gate, x, state, lengths,
  reverse)`, or with the factors and the addends themselves, `lax.linear_recurrence(factor, x, state, lengths, reverse)`.

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
EPS = 1e-5


# ------------------------------------------------------------------ the cases

def listed():
    return [
        #the last features of one image that is served: the smallest call, latency only
        dict(name='group_norm_image', op='group_norm', way='forward', batch=1, height=7, width=7, channels=512, groups=32, activation='silu'),
        #one normalisation in the middle of a convolutional network
        dict(name='group_norm_block_32', op='group_norm', way='forward', batch=32, height=56, width=56, channels=64, groups=32, activation='relu'),
        #a training step's widest normalisation in a deep network, forward and backward
        dict(name='group_norm_train_64', op='group_norm', way='train', batch=64, height=56, width=56, channels=256, groups=32, activation='relu'),
        #heads of a token model normalised position by position, odd number of positions and of channels in a group
        dict(name='group_norm_heads', op='group_norm', way='train', batch=8191, height=1, width=1, channels=1040, groups=16, activation='silu'),
        #a served batch of eight sequences: the sampled tokens' log probabilities with the twenty most likely alternatives; some of
        #the vocabulary is masked
        dict(name='log_probs_decode', op='token_log_probs', way='forward', rows=8, vocabulary=32000, top=20, padded=0, masked=True),
        #a classifier's scores over many samples: the labels' log probabilities, the doubt, and the five best classes
        dict(name='log_probs_classes', op='token_log_probs', way='forward', rows=65536, vocabulary=1000, top=5, padded=0, masked=False),
        #a training step's loss over a vocabulary, some positions padded
        dict(name='log_probs_train', op='token_log_probs', way='train', rows=4096, vocabulary=32000, top=0, padded=256, masked=False),
        #the same with odd sizes, and fewer rows than fill the machine several times over
        dict(name='log_probs_ragged', op='token_log_probs', way='train', rows=321, vocabulary=50001, top=3, padded=7, masked=True),
        #one token of each of 64 sequences that are decoded together
        dict(name='recurrence_token', op='recurrence', way='forward', gated=True, batch=64, time=1, channels=2048, state=True, ragged=False, reverse=False),
        #a long document read at once: one sequence, few channels
        dict(name='recurrence_long', op='recurrence', way='forward', gated=True, batch=1, time=65536, channels=1024, state=True, ragged=False, reverse=False),
        #a training step over a padded batch
        dict(name='recurrence_train', op='recurrence', way='train', gated=True, batch=8, time=2048, channels=2048, state=True, ragged=True, reverse=False),
        #factors and addends of the model's own, backwards in time, odd sizes
        dict(name='recurrence_ragged', op='recurrence', way='train', gated=False, batch=3, time=1021, channels=333, state=False, ragged=True, reverse=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def _width(rng, low, high):
    '''A number of channels: mostly a multiple of 8, at times any number.'''
    n = _log_int(rng, low, high)
    return n if rng.random() < 0.3 else max(low, n // 8 * 8)


def draw(rng):
    op = rng.choice(('group_norm', 'token_log_probs', 'recurrence'))
    case = dict(op=op, way=rng.choice(('forward', 'train')))
    if op == 'group_norm':
        groups = rng.choice((1, 2, 3, 4, 8, 16, 32, 32, 64))
        #(groups of at least 16 values: what is normalised over one or two is all but constant, and its gradient a rounding)
        if rng.random() < 0.3:
            channels, height, width = groups * _log_int(rng, 16, max(16, 2048 // groups)), 1, 1
        else:
            channels, height, width = groups * _log_int(rng, 1, max(1, 2048 // groups)), _log_int(rng, 4, 112), _log_int(rng, 4, 112)
        most = max(1, int(51e6 // (height * width * channels)))
        case.update(batch=_log_int(rng, 1, min(most, 128 if height > 1 else 16384)), height=height, width=width, channels=channels,
                    groups=groups, activation=rng.choice(('none', 'relu', 'silu')))
    elif op == 'token_log_probs':
        vocabulary = _log_int(rng, 10, 262144)
        rows = _log_int(rng, 1, max(1, min(65536, int(131e6 // vocabulary))))
        case.update(rows=rows, vocabulary=vocabulary, top=rng.choice((0, 0, 1, 5, 8, 20, 32)), padded=rng.choice((0, rows // 8)),
                    masked=rng.random() < 0.3)
        case['top'] = min(case['top'], vocabulary)
    else:
        channels = _width(rng, 8, 4096)
        time = rng.choice((1, _log_int(rng, 2, 65536), _log_int(rng, 2, 65536)))
        most = max(1, int((67e6 if case['way'] == 'forward' else 33e6) // (time * channels)))
        if time * channels > 33e6:
            channels = max(8, int(33e6 // time))
        case.update(batch=_log_int(rng, 1, min(64, most)), time=time, channels=channels, gated=rng.random() < 0.6,
                    state=rng.random() < 0.5, ragged=rng.random() < 0.5, reverse=rng.random() < 0.25)
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

    if case['op'] == 'group_norm':
        #what a convolution leaves: channels with an offset and a spread of their own
        c, shape = case['channels'], (case['batch'], case['height'], case['width'], case['channels'])
        x = normal(*shape).mul_(0.5 + uniform(c)).add_(normal(c, scale=0.5))
        found = dict(x=x, scale=0.5 + uniform(c), shift=normal(c, scale=0.1))
        if case['way'] == 'train':
            found['g'] = normal(*shape)
        return found
    if case['op'] == 'token_log_probs':
        #scores whose best ones stand out; padded positions hold the token -1
        rows, v = case['rows'], case['vocabulary']
        logits = normal(rows, v, scale=2.0)
        tokens = integers(v, rows)
        logits.scatter_add_(1, tokens.long()[:, None], 6.0 * uniform(rows, 1))
        if case['masked']:
            #a part of the vocabulary is not allowed here; the given token is
            barred = uniform(rows, v) < 0.25
            barred.scatter_(1, tokens.long()[:, None], False)
            #(as many as are asked for stay allowed)
            barred[:, :max(1, case['top'])] = False
            logits.masked_fill_(barred, float('-inf'))
        if case['padded']:
            tokens[torch.randperm(rows, generator=g, device=DEVICE)[:case['padded']]] = -1
        found = dict(logits=logits, tokens=tokens)
        if case['way'] == 'train':
            #a mean over the rows, and a reward for entropy
            found['g_log_probs'] = normal(rows, scale=1.0 / rows)
            found['g_entropy'] = normal(rows, scale=0.1 / rows)
            if case['top']:
                found['g_top'] = normal(rows, case['top'], scale=1.0 / rows)
        return found
    b, t, c = case['batch'], case['time'], case['channels']
    if case['gated']:
        found = dict(gate=normal(b, t, c, scale=1.5, shift=2.0), x=normal(b, t, c))
    else:
        found = dict(gate=1.0 - 0.3 * uniform(b, t, c), x=normal(b, t, c, scale=0.5))
    if case['state']:
        found['state'] = normal(b, c)
    if case['ragged']:
        found['lengths'] = torch.tensor(_lengths(case, int(integers(b, 1).item())), dtype=torch.int32, device=DEVICE)
    if case['way'] == 'train':
        found['g'], found['g_last'] = normal(b, t, c), normal(b, c)
    return found


# ------------------------------------------------------------------ the framework's programs

class _InHBM:
    '''A result array of a recorded program where it lies in HBM.'''
    def __init__(self, buffer):
        kind = '<f4' if buffer.dtype == np.float32 else '<i4'
        self.owner = buffer
        self.__cuda_array_interface__ = dict(shape=buffer.shape, typestr=kind, data=(buffer.tensor.device_ptr(), False), version=2)


def _program(case, names):
    '''A function of the arrays `names` for the framework to trace.'''
    from vkjax_amd import minijax as mj
    nn, lax = mj.nn, mj.lax
    if case['op'] == 'group_norm':
        activation = None if case['activation'] == 'none' else case['activation']

        def norm(x, scale, shift):
            return nn.group_norm(x, scale, shift, case['groups'], eps=EPS, activation=activation)

        def train(x, scale, shift, g):
            y, pullback = mj.vjp(norm, x, scale, shift)
            return (y,) + tuple(pullback(g))
        return norm if case['way'] == 'forward' else train
    if case['op'] == 'token_log_probs':
        def log_probs(logits, tokens):
            return nn.token_log_probs(logits, tokens, top=case['top'])

        def train(logits, tokens, *cotangents):
            if case['top']:
                #(the alternatives' tokens have no gradient)
                def split(z):
                    outs = log_probs(z, tokens)
                    return outs[:3], outs[3]
                outs, pullback, top_tokens = mj.vjp(split, logits, has_aux=True)
                return tuple(outs) + (top_tokens,) + tuple(pullback(tuple(cotangents)))
            outs, pullback = mj.vjp(lambda z: log_probs(z, tokens), logits)
            return tuple(outs) + tuple(pullback(tuple(cotangents)))
        return log_probs if case['way'] == 'forward' else train

    def forward(a):
        f = nn.gated_recurrence if case['gated'] else lax.linear_recurrence
        return f(a['gate'], a['x'], a.get('state'), a.get('lengths'), reverse=case['reverse'])

    def recurrence(*arrays):
        return forward(dict(zip(names, arrays)))

    def train_recurrence(*arrays):
        a = dict(zip(names, arrays))
        wrt = [n for n in ('gate', 'x', 'state') if n in a]
        outs, pullback = mj.vjp(lambda *values: forward(dict(a, **dict(zip(wrt, values)))), *[a[n] for n in wrt])
        return tuple(outs) + tuple(pullback((a['g'], a['g_last'])))
    return recurrence if case['way'] == 'forward' else train_recurrence


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
    case, a = state['case'], state['arrays']
    return {'group_norm': _plain_group_norm, 'token_log_probs': _plain_log_probs, 'recurrence': _plain_recurrence}[case['op']](case, **a)


# ------------------------------------------------------------------ the plain forms

def _plain_group_norm(case, x, scale, shift, g=None):
    n, c, groups = x.shape[0], x.shape[-1], case['groups']
    by_group = lambda v: v.reshape(n, -1, groups, c // groups)
    xg = by_group(x)
    centred = xg - xg.mean(dim=(1, 3), keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + EPS)
    hat = centred * rstd
    gamma, beta = scale.reshape(groups, -1), shift.reshape(groups, -1)
    z = hat * gamma + beta
    gate = None
    if case['activation'] == 'relu':
        y = torch.where(z > 0, z, torch.zeros_like(z))
    elif case['activation'] == 'silu':
        gate = 1.0 / (1.0 + torch.exp(-z))
        y = z * gate
    else:
        y = z
    if g is None:
        return [y.reshape(x.shape)]
    d = by_group(g)
    if case['activation'] == 'relu':
        d = torch.where(z > 0, d, torch.zeros_like(d))
    elif case['activation'] == 'silu':
        d = d * (gate * (1.0 + z * (1.0 - gate)))
    dshift, dscale = d.sum(dim=(0, 1)), (d * hat).sum(dim=(0, 1))
    d = d * gamma
    dx = rstd * (d - d.mean(dim=(1, 3), keepdim=True) - hat * (d * hat).mean(dim=(1, 3), keepdim=True))
    return [y.reshape(x.shape), dx.reshape(x.shape), dscale.reshape(-1), dshift.reshape(-1)]


def _plain_log_probs(case, logits, tokens, g_log_probs=None, g_entropy=None, g_top=None):
    v, top = logits.shape[1], case['top']
    given = (tokens >= 0) & (tokens < v)
    at = torch.where(given, tokens, torch.zeros_like(tokens)).long()[:, None]
    best = logits.max(dim=1, keepdim=True).values
    log_sum = best + torch.log(torch.exp(logits - best).sum(dim=1, keepdim=True))
    logp = logits - log_sum
    p = torch.exp(logp)
    zero = torch.zeros((), device=logits.device)
    entropy = -torch.where(p > 0, p * logp, zero).sum(dim=1)
    outs = [torch.where(given, logp.gather(1, at)[:, 0], zero), torch.where(given, entropy, zero)]
    if top:
        #(equal scores by their place: a stable sort)
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
        outs.append(torch.where(given[:, None], logp.gather(1, order), zero))
        outs.append(torch.where(given[:, None], order.int(), torch.full_like(order, -1, dtype=torch.int32)))
    if g_log_probs is None:
        return outs
    d = torch.where(p > 0, p * (logp + entropy[:, None]), zero) * -g_entropy[:, None]
    total = g_log_probs if g_top is None else g_log_probs + g_top.sum(dim=1)
    d = d - p * total[:, None]
    d = d.scatter_add(1, at, g_log_probs[:, None])
    if g_top is not None:
        d = d.scatter_add(1, order, g_top)
    return outs + [torch.where(given[:, None], d, zero)]


def _scan(a, b):
    '''h[t] = a[t] h[t-1] + b[t] along axis 1 from h[-1] = 0, by doubling.'''
    a, h, step = a.clone(), b.clone(), 1
    while step < h.shape[1]:
        h[:, step:] = h[:, step:] + a[:, step:] * h[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return h


def _plain_recurrence(case, gate, x, state=None, lengths=None, g=None, g_last=None):
    t = x.shape[1]
    a = 1.0 / (1.0 + torch.exp(-gate)) if case['gated'] else gate
    b = (1.0 - a) * x if case['gated'] else x
    inside = None
    if lengths is not None:
        #positions behind a sequence's end keep the state
        inside = torch.arange(t, device=x.device)[None, :, None] < lengths[:, None, None]
        a = torch.where(inside, a, torch.ones_like(a))
        b = torch.where(inside, b, torch.zeros_like(b))
    turn = (lambda v: v.flip(1)) if case['reverse'] else (lambda v: v)
    first = torch.zeros_like(x[:, 0]) if state is None else state
    start = turn(b).clone()
    start[:, 0] = start[:, 0] + turn(a)[:, 0] * first
    h = _scan(turn(a), start)
    last = h[:, -1].clone()
    outs = [turn(h), last]
    if g is None:
        return outs
    #the adjoint runs the other way: l[t] = g[t] + a[t+1] l[t+1]
    ta = turn(a)
    back = torch.cat([ta[:, 1:], torch.ones_like(ta[:, :1])], dim=1).flip(1)
    seeds = turn(g).clone()
    seeds[:, -1] = seeds[:, -1] + g_last
    adjoint = _scan(back, seeds.flip(1)).flip(1)
    before = torch.cat([first[:, None], h[:, :-1]], dim=1)
    dstate = ta[:, 0] * adjoint[:, 0]
    adjoint, before = turn(adjoint), turn(before)
    if case['gated']:
        dgate, dx = adjoint * (before - x) * a * (1.0 - a), adjoint * (1.0 - a)
    else:
        dgate, dx = adjoint * before, adjoint
    if inside is not None:
        dgate, dx = torch.where(inside, dgate, torch.zeros_like(dgate)), torch.where(inside, dx, torch.zeros_like(dx))
    return outs + [dgate, dx] + ([dstate] if state is not None else [])


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    a = {k: v.double() if v.dtype == torch.float32 else v for k, v in _inputs(case, seed).items()}
    return {'group_norm': _exact_group_norm, 'token_log_probs': _exact_log_probs, 'recurrence': _exact_recurrence}[case['op']](case, **a)


def _exact_group_norm(case, x, scale, shift, g=None):
    outs = ([], [])
    groups, c = case['groups'], case['channels']
    dscale, dshift = torch.zeros_like(scale), torch.zeros_like(shift)
    for i in range(0, x.shape[0], 1024 if x[0].numel() < 1 << 14 else 8):          #a few samples at a time: 64 bits take room
        part = slice(i, i + (1024 if x[0].numel() < 1 << 14 else 8))
        v = x[part]
        n = v.shape[0]
        cut = v.reshape(n, -1, groups, c // groups).transpose(1, 2).reshape(n, groups, -1)
        var, mean = torch.var_mean(cut, dim=2, correction=0)
        spread = lambda s: s.repeat_interleave(c // groups, dim=1)[:, None, None, :]
        inv = spread(1.0 / torch.sqrt(var + EPS))
        hat = (v - spread(mean)) * inv
        z = hat * scale + shift
        act = case['activation']
        y = z.clamp(min=0) if act == 'relu' else z * torch.sigmoid(z) if act == 'silu' else z
        outs[0].append(y)
        if g is None:
            continue
        d = g[part]
        if act == 'relu':
            d = d * (z > 0)
        elif act == 'silu':
            s = torch.sigmoid(z)
            d = d * (s + z * s * (1 - s))
        dshift += d.sum(dim=(0, 1, 2))
        dscale += (d * hat).sum(dim=(0, 1, 2))
        d = d * scale
        size = cut.shape[2]
        over = lambda s: spread(s.sum(dim=(1, 2)).reshape(n, groups, -1).sum(dim=2) / size)
        outs[1].append(inv * (d - over(d) - hat * over(d * hat)))
    found = [torch.cat(outs[0])]
    return found if g is None else found + [torch.cat(outs[1]), dscale, dshift]


def _exact_log_probs(case, logits, tokens, g_log_probs=None, g_entropy=None, g_top=None):
    found, top, v = [], case['top'], case['vocabulary']
    step = max(1, (1 << 25) // v)
    for i in range(0, logits.shape[0], step):
        part = slice(i, i + step)
        z, token = logits[part], tokens[part].long()
        keep = (token >= 0) & (token < v)
        token = token.clamp(0, v - 1)
        logp = torch.log_softmax(z, dim=1)
        p = logp.exp()
        finite = logp.masked_fill(p == 0, 0.0)
        entropy = -(p * finite).sum(dim=1)
        rows = torch.arange(z.shape[0], device=z.device)
        outs = [logp[rows, token] * keep, entropy * keep]
        if top:
            #(-score, place) in rising order
            best = torch.argsort(-z, dim=1, stable=True)[:, :top]
            outs += [torch.gather(logp, 1, best).masked_fill(~keep[:, None], 0.0), best.masked_fill(~keep[:, None], -1).int()]
        if g_log_probs is not None:
            d = -g_entropy[part, None] * p * (finite + entropy[:, None]) - p * g_log_probs[part, None]
            d[rows, token] += g_log_probs[part]
            if g_top is not None:
                for j in range(top):
                    d -= p * g_top[part, j, None]
                    d[rows, best[:, j]] += g_top[part, j]
            outs.append(d * keep[:, None])
        found.append(outs)
    return [torch.cat(parts) for parts in zip(*found)]


def _exact_recurrence(case, gate, x, state=None, lengths=None, g=None, g_last=None):
    t = x.shape[1]
    a = torch.sigmoid(gate) if case['gated'] else gate.clone()
    u = (1 - a) * x if case['gated'] else x.clone()
    if lengths is not None:
        for i, n in enumerate(lengths.tolist()):
            a[i, n:], u[i, n:] = 1.0, 0.0
    order = range(t - 1, -1, -1) if case['reverse'] else range(t)
    h, first = torch.empty_like(x), torch.zeros_like(x[:, 0]) if state is None else state
    now = first
    for k in order:
        torch.addcmul(u[:, k], a[:, k], now, out=h[:, k])
        now = h[:, k]
    outs = [h, now.clone()]
    if g is None:
        return outs
    da, du, adjoint = torch.empty_like(x), torch.empty_like(x), g_last.clone()
    steps = list(order)
    for place in range(t - 1, -1, -1):
        k = steps[place]
        adjoint += g[:, k]
        du[:, k] = adjoint
        torch.mul(adjoint, h[:, steps[place - 1]] if place else first, out=da[:, k])
        adjoint *= a[:, k]
    if case['gated']:
        dgate, dx = (da - du * x) * a * (1 - a), du * (1 - a)
    else:
        dgate, dx = da, du
    if lengths is not None:
        for i, n in enumerate(lengths.tolist()):
            dgate[i, n:], dx[i, n:] = 0.0, 0.0
    return outs + [dgate, dx] + ([adjoint] if state is not None else [])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    train = case['way'] == 'train'
    if case['op'] == 'group_norm':
        n = case['batch'] * case['height'] * case['width'] * case['channels']
        return dict(bytes=4 * (n * (4 if train else 2) + case['channels'] * (4 if train else 2)), flops=n * (24 if train else 9))
    if case['op'] == 'token_log_probs':
        rows, v, given = case['rows'], case['vocabulary'], case['rows'] - case['padded']
        small = rows * (3 + 2 * case['top']) + (rows * (2 + case['top']) if train else 0)
        return dict(bytes=4 * (given * v + (rows * v if train else 0) + small), flops=given * v * (12 if train else 6))
    b, t, c = case['batch'], case['time'], case['channels']
    n, inside = b * t * c, c * (sum(_lengths(case)) if case['ragged'] else b * t)
    rows = b * c * (1 + case['state'])
    if not train:
        return dict(bytes=4 * (2 * inside + n + rows), flops=inside * (8 if case['gated'] else 2))
    return dict(bytes=4 * (2 * inside + n + 3 * n + rows * 2), flops=inside * (20 if case['gated'] else 6))
