"""What the sequence operators are measured on: the parts of a state space block between its matrix products.

Three operators, each in the forms a user's program calls: the selective scan and the short causal convolution over
prompts, for training (forward and backward) and for single tokens with a kept state; the root-mean-square norm that
adds the residual, for training and with an 8-bit output.  With ``own`` false a pass computes the plain form from
elementary torch operations, with ``own`` true it calls the framework.
"""
import math

import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
SIZE = {'bf16': 2, 'fp16': 2, 'fp32': 4}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------
# cases

def _scan(name, dtype, batch, length, channels, states, groups=1, ragged=False, train=False):
    return {'name': name, 'op': 'scan', 'dtype': dtype, 'batch': batch, 'length': length, 'channels': channels,
            'states': states, 'groups': groups, 'ragged': ragged, 'train': train}


def _scan_step(name, dtype, batch, channels, states, groups=1):
    return {'name': name, 'op': 'scan_step', 'dtype': dtype, 'batch': batch, 'channels': channels, 'states': states,
            'groups': groups}


def _conv(name, dtype, batch, length, channels, taps, ragged=False, train=False):
    return {'name': name, 'op': 'conv', 'dtype': dtype, 'batch': batch, 'length': length, 'channels': channels,
            'taps': taps, 'ragged': ragged, 'train': train}


def _conv_step(name, dtype, batch, channels, taps):
    return {'name': name, 'op': 'conv_step', 'dtype': dtype, 'batch': batch, 'channels': channels, 'taps': taps}


def _norm(name, dtype, rows, columns, residual=True, train=False):
    return {'name': name, 'op': 'norm', 'dtype': dtype, 'rows': rows, 'columns': columns, 'residual': residual,
            'train': train}


def _quantize(name, dtype, rows, columns, group, residual=True):
    return {'name': name, 'op': 'quantize', 'dtype': dtype, 'rows': rows, 'columns': columns, 'group': group,
            'residual': residual}


def listed():
    return [
        # one conversation that is answered token by token: latency is all
        _scan_step('scan step 1', 'bf16', 1, 2048, 16),
        # a full serving batch, one token each: the states are read and written
        _scan_step('scan step 256', 'bf16', 256, 4096, 16),
        # an ordinary prompt of one user
        _scan('scan prompt 2k', 'bf16', 1, 2048, 2048, 16),
        # a long document in one piece
        _scan('scan prompt 16k', 'bf16', 1, 16384, 4096, 16),
        # a training step of ordinary sizes
        _scan('scan train', 'bf16', 4, 2048, 2048, 16, train=True),
        # training in full precision on a padded batch of sequences of odd sizes, two groups of channels
        _scan('scan train odd', 'fp32', 3, 777, 650, 24, groups=2, ragged=True, train=True),
        # one token each of a serving batch
        _conv_step('conv step 64', 'bf16', 64, 4096, 4),
        # prompts of several users, padded, odd sizes
        _conv('conv prompt odd', 'fp16', 5, 1777, 1030, 3, ragged=True),
        # a training step
        _conv('conv train', 'bf16', 4, 4096, 4096, 4, train=True),
        # a training step: the residual stream of 16384 tokens
        _norm('norm train', 'bf16', 16384, 4096, train=True),
        # tokens on their way into a matrix product in 8 bits: a scale per 128 columns
        _quantize('norm to 8 bits', 'bf16', 16384, 4096, 128),
        # the same for a few tokens that are decoded: one scale per row
        _quantize('norm to 8 bits, 8 rows', 'bf16', 8, 2048, 0),
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['scan', 'scan', 'scan', 'scan_step', 'conv', 'conv', 'conv_step', 'norm', 'quantize'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if op in ('scan', 'scan_step'):
        groups = rng.choice([1, 1, 1, 2, 4])
        states = rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 128)])
        if op == 'scan_step':
            return _without_name(_scan_step('', dtype, _log(rng, 1, 256), groups * _log(rng, 16, 4096 // groups), states,
                                            groups))
        train = rng.random() < 0.5
        most = (1 << 28) if train else (1 << 30)
        batch, channels = _log(rng, 1, 8), groups * _log(rng, 16, 4096 // groups)
        length = _log(rng, 1, max(1, min(16384, most // (batch * channels * states))))
        return _without_name(_scan('', dtype, batch, length, channels, states, groups, rng.random() < 0.4, train))
    if op == 'conv_step':
        return _without_name(_conv_step('', dtype, _log(rng, 1, 256), _log(rng, 16, 8192), rng.randint(2, 8)))
    if op == 'conv':
        batch, channels = _log(rng, 1, 8), _log(rng, 16, 8192)
        length = _log(rng, 1, max(1, min(16384, (1 << 26) // (batch * channels))))
        return _without_name(_conv('', dtype, batch, length, channels, rng.choice([4, 4, 2, 3, rng.randint(1, 8)]),
                                   rng.random() < 0.4, rng.random() < 0.5))
    columns = rng.choice([_log(rng, 16, 16384), 128 * rng.randint(1, 64)])
    rows = _log(rng, 1, max(1, min(32768, (1 << 26) // columns)))
    if op == 'norm':
        return _without_name(_norm('', dtype, rows, columns, rng.random() < 0.7, rng.random() < 0.5))
    return _without_name(_quantize('', dtype, rows, columns, 128 if columns % 128 == 0 and rng.random() < 0.6 else 0,
                                   rng.random() < 0.7))


def _without_name(case):
    del case['name']
    return case


# ---------------------------------------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    t = TYPES[case['dtype']]

    def normal(*shape, scale=1.0, dtype=t):
        return torch.empty(shape, device='cuda').normal_(0, scale, generator=gen).to(dtype)

    s = {'case': dict(case)}
    op = case['op']
    if op in ('scan', 'scan_step'):
        b, d, n, g = case['batch'], case['channels'], case['states'], case['groups']
        lead = (b,) if op == 'scan_step' else (b, case['length'])
        # u and z are the halves of one projection, delta, B and C come out of others: views with the strides of the whole
        both = normal(*lead, 2 * d)
        s['u'], s['z'] = both[..., :d], both[..., d:]
        bc = normal(*lead, 2 * g * n)
        s['B'], s['C'] = bc[..., :g * n].unflatten(-1, (g, n)), bc[..., g * n:].unflatten(-1, (g, n))
        s['delta'] = normal(*lead, d, scale=0.5)
        # decays from 1 to the number of states, step sizes spread over 0.001 to 0.1: as such layers are initialised
        s['A'] = -torch.arange(1, n + 1, device='cuda', dtype=torch.float32).repeat(d, 1)
        s['A'] *= torch.empty(d, n, device='cuda').uniform_(0.9, 1.1, generator=gen)
        step = torch.exp(torch.empty(d, device='cuda').uniform_(math.log(1e-3), math.log(1e-1), generator=gen))
        s['delta_bias'] = step + torch.log(-torch.expm1(-step))
        s['D'] = normal(d, dtype=torch.float32)
        s['state'] = normal(b, d, n, scale=0.5, dtype=torch.float32)
        if op == 'scan':
            s['lengths'] = None
            if case['ragged']:
                s['lengths'] = torch.randint(0, case['length'] + 1, (b,), device='cuda', generator=gen, dtype=torch.int32)
            if case['train']:
                s['gout'] = normal(b, case['length'], d)
                s['gstate'] = normal(b, d, n, dtype=torch.float32)
    elif op in ('conv', 'conv_step'):
        b, d, w = case['batch'], case['channels'], case['taps']
        lead = (b,) if op == 'conv_step' else (b, case['length'])
        s['x'] = normal(*lead, 2 * d)[..., :d]
        s['weight'] = normal(d, w, scale=w ** -0.5)
        s['bias'] = normal(d, scale=0.1)
        s['state'] = normal(b, w - 1, d)
        if op == 'conv':
            s['lengths'] = None
            if case['ragged']:
                s['lengths'] = torch.randint(0, case['length'] + 1, (b,), device='cuda', generator=gen, dtype=torch.int32)
            if case['train']:
                s['gout'] = normal(b, case['length'], d)
                s['gstate'] = normal(b, w - 1, d)
    else:
        shape = (case['rows'], case['columns'])
        s['x'] = normal(*shape)
        s['residual'] = normal(*shape, scale=2.0) if case['residual'] else None
        s['weight'] = (1 + 0.1 * torch.empty(shape[1], device='cuda').normal_(0, 1, generator=gen)).to(t)
        if case.get('train'):
            s['gout'] = normal(*shape)
            s['gres'] = normal(*shape) if case['residual'] else None
    if case.get('train'):
        for k in _leaves(op):
            if s[k] is not None:
                s[k] = s[k].detach().requires_grad_()
    return s


def _leaves(op):
    return {'scan': ('u', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias', 'state'),
            'conv': ('x', 'weight', 'bias', 'state'), 'norm': ('x', 'residual', 'weight')}[op]


# ---------------------------------------------------------------------------------------------------------
# the calls of the framework

def _own(s):
    import opveclib_b200 as ovl
    case = s['case']
    op = case['op']
    if op == 'scan_step':
        out = ovl.selective_scan_step(s['state'], s['u'], s['delta'], s['A'], s['B'], s['C'], s['D'], s['z'],
                                      s['delta_bias'], delta_softplus=True)
        return [out, s['state']]
    if op == 'conv_step':
        out = ovl.causal_conv1d_step(s['state'], s['x'], s['weight'], s['bias'], activation='silu')
        return [out, s['state']]
    if op == 'quantize':
        return list(ovl.rms_norm_quantize(s['x'], s['weight'], s['residual'], eps=EPS, group=case['group'] or None))
    if op == 'scan':
        outs = ovl.selective_scan(s['u'], s['delta'], s['A'], s['B'], s['C'], s['D'], s['z'], s['delta_bias'],
                                  delta_softplus=True, initial_state=s['state'], lengths=s['lengths'], return_state=True)
    elif op == 'conv':
        outs = ovl.causal_conv1d(s['x'], s['weight'], s['bias'], activation='silu', initial_state=s['state'],
                                 lengths=s['lengths'], return_state=True)
    else:
        outs = ovl.rms_norm(s['x'], s['weight'], s['residual'], eps=EPS)
        outs = outs if isinstance(outs, tuple) else (outs,)
    if not case['train']:
        return list(outs)
    above = [s['gout'], s['gres'] if op == 'norm' else s['gstate']][:len(outs)]
    grads = torch.autograd.grad(outs, [s[k] for k in _leaves(op) if s[k] is not None], above)
    return [o.detach() for o in outs] + list(grads)


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {'scan': _plain_scan, 'scan_step': _plain_scan_step, 'conv': _plain_conv, 'conv_step': _plain_conv_step,
                'norm': _plain_norm, 'quantize': _plain_quantize}[s['case']['op']](s)


# ---------------------------------------------------------------------------------------------------------
# the plain forms: 32 bits, rounded once at the end

def _inside(lengths, length):
    """Which tokens belong to their sequence, [batch, length, 1]; all of them where no lengths are given."""
    at = torch.arange(length, device='cuda')[None, :, None]
    return at < (length if lengths is None else lengths.long()[:, None, None])


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp(max=20))))


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1, in place in b: after step k every h_t holds its last 2^k terms."""
    s = 1
    while s < b.shape[1]:
        b[:, s:] = b[:, s:] + a[:, s:] * b[:, :-s]
        a[:, s:] = a[:, s:] * a[:, :-s]
        s *= 2
    return b


def _plain_scan(s):
    case = s['case']
    t, g, length = TYPES[case['dtype']], case['groups'], case['length']
    inside = _inside(s['lengths'], length)

    def split(x):                                            # channels -> groups x channels of a group
        return x.unflatten(2, (g, -1))

    u = torch.where(inside, s['u'].float(), 0.0)
    z = torch.where(inside, s['z'].float(), 0.0)
    raw = s['delta'].float() + s['delta_bias']
    dt = torch.where(inside, _softplus(raw), 0.0)
    A = s['A'].unflatten(0, (g, -1))
    B = torch.where(inside[..., None], s['B'].float(), 0.0).unsqueeze(3)
    C = torch.where(inside[..., None], s['C'].float(), 0.0).unsqueeze(3)
    h0 = s['state'].unflatten(1, (g, -1))
    a = torch.exp(split(dt)[..., None] * A)
    h = split(dt * u)[..., None] * B
    h[:, 0] += a[:, 0] * h0
    h = _recurrence(a, h)
    y = (h * C).sum(-1).flatten(2) + s['D'] * u
    sig = torch.sigmoid(z)
    out = torch.where(inside, y * z * sig, 0.0).to(t)
    final = h[:, -1].flatten(1, 2).clone()
    if not case['train']:
        return [out, final]
    gout = torch.where(inside, s['gout'].float(), 0.0)
    gy = gout * z * sig
    gz = gout * y * (sig + z * sig * (1 - sig))
    # the recurrence of the gradient runs backwards: gh_t = C_t gy_t + a_{t+1} gh_{t+1}
    torch.exp(split(dt)[..., None] * A, out=a)
    gh = split(gy)[..., None] * C
    gh[:, -1] += s['gstate'].unflatten(1, (g, -1))
    after = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    gh = _recurrence(after, gh.flip(1)).flip(1)
    del after
    gC = torch.where(inside[..., None], (split(gy)[..., None] * h).sum(3), 0.0)
    gB = (gh * split(dt * u)[..., None]).sum(3)
    q = a * gh
    gh0 = q[:, 0].flatten(1, 2).clone()
    q[:, 1:] *= h[:, :-1]
    q[:, 0] *= h0
    gA = (q * split(dt)[..., None]).sum((0, 1)).flatten(0, 1)
    over = (gh * B).sum(-1).flatten(2)
    gdt = (q * A).sum(-1).flatten(2) + u * over
    gu = dt * over + s['D'] * gy
    graw = torch.where(inside, gdt * torch.sigmoid(raw), 0.0)
    return [out, final, gu.to(t), graw.to(t), gA, gB.to(t), gC.to(t), (gy * u).sum((0, 1)), gz.to(t),
            graw.sum((0, 1)), gh0]


def _plain_scan_step(s):
    case = s['case']
    g = case['groups']
    u, z = s['u'].float(), s['z'].float()
    dt = _softplus(s['delta'].float() + s['delta_bias'])
    h = s['state'].unflatten(1, (g, -1))
    new = torch.exp(dt[..., None] * s['A']).unflatten(1, (g, -1)) * h
    new += (dt * u).unflatten(1, (g, -1))[..., None] * s['B'].float()[:, :, None]
    s['state'].copy_(new.flatten(1, 2))
    y = (new * s['C'].float()[:, :, None]).sum(-1).flatten(1) + s['D'] * u
    return [(y * z * torch.sigmoid(z)).to(TYPES[case['dtype']]), s['state']]


def _plain_conv(s):
    case = s['case']
    t, length, taps = TYPES[case['dtype']], case['length'], case['taps']
    inside = _inside(s['lengths'], length)
    w, bias = s['weight'].float(), s['bias'].float()
    x = torch.cat([s['state'].float(), torch.where(inside, s['x'].float(), 0.0)], 1)
    windows = x.unfold(1, taps, 1)                           # [batch, length, channels, taps]
    pre = (windows * w).sum(-1) + bias
    sig = torch.sigmoid(pre)
    out = torch.where(inside, pre * sig, 0.0).to(t)
    # the state after a sequence: its last taps - 1 inputs, those before it among them
    end = torch.full((case['batch'],), length, device='cuda') if s['lengths'] is None else s['lengths'].long()
    last = (end[:, None] + torch.arange(taps - 1, device='cuda'))[..., None].expand(-1, -1, case['channels'])
    final = x.gather(1, last).to(t)
    if not case['train']:
        return [out, final]
    gpre = torch.where(inside, s['gout'].float() * (sig + pre * sig * (1 - sig)), 0.0)
    padded = torch.nn.functional.pad(gpre, (0, 0, taps - 1, taps - 1))
    gx = (padded.unfold(1, taps, 1) * w.flip(1)).sum(-1)
    gx.scatter_add_(1, last, s['gstate'].float())
    gw = (gpre[..., None] * windows).sum((0, 1))
    return [out, final, gx[:, taps - 1:].to(t), gw.to(t), gpre.sum((0, 1)).to(t), gx[:, :taps - 1].to(t)]


def _plain_conv_step(s):
    x = torch.cat([s['state'], s['x'][:, None]], 1)
    pre = (x.float() * s['weight'].float().t()).sum(1) + s['bias'].float()
    s['state'].copy_(x[:, 1:])
    return [(pre * torch.sigmoid(pre)).to(TYPES[s['case']['dtype']]), s['state']]


def _normed(s):
    x = s['x'].float() if s['residual'] is None else s['x'].float() + s['residual'].float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x, r, x * r * s['weight'].float()


def _plain_norm(s):
    t = TYPES[s['case']['dtype']]
    x, r, y = _normed(s)
    outs = [y.to(t)] if s['residual'] is None else [y.to(t), x.to(t)]
    if not s['case']['train']:
        return outs
    xhat, gy = x * r, s['gout'].float()
    g = gy * s['weight'].float()
    gx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    if s['residual'] is not None:
        gx += s['gres'].float()
    gx = gx.to(t)
    return outs + [gx] * len(outs) + [(gy * xhat).sum(0).to(t)]


def _plain_quantize(s):
    x, r, y = _normed(s)
    parts = y.unflatten(-1, (-1, s['case']['group'] or s['case']['columns']))
    scale = (parts.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
    q = (parts / scale[..., None]).flatten(-2).to(torch.float8_e4m3fn)
    return [q, scale] if s['residual'] is None else [q, scale, x.to(TYPES[s['case']['dtype']])]


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    e, op = SIZE[case['dtype']], case['op']
    if op in ('scan', 'scan_step'):
        b, d, n = case['batch'], case['channels'], case['states']
        tokens = b * case.get('length', 1)
        vectors, bc, state = tokens * d * e, tokens * case['groups'] * n * e, b * d * n * 4
        params = d * n * 4 + 2 * d * 4
        if not case.get('train'):
            return {'bytes': 4 * vectors + 2 * bc + 2 * state + params, 'flops': tokens * d * (7 * n + 10)}
        # forward: u, delta, z, out; backward: u, delta, z, gout and the gradients of the first three
        return {'bytes': 11 * vectors + 6 * bc + 5 * state + 3 * params, 'flops': tokens * d * (28 * n + 40)}
    if op in ('conv', 'conv_step'):
        b, d, w = case['batch'], case['channels'], case['taps']
        vectors, state = b * case.get('length', 1) * d, b * (w - 1) * d
        if not case.get('train'):
            return {'bytes': (2 * vectors + 2 * state + d * (w + 1)) * e, 'flops': vectors * (2 * w + 6)}
        return {'bytes': (5 * vectors + 5 * state + 3 * d * (w + 1)) * e, 'flops': vectors * (8 * w + 20)}
    values, more = case['rows'] * case['columns'], 2 if case['residual'] else 0
    if op == 'quantize':
        scales = case['rows'] * (case['columns'] // case['group'] if case['group'] else 1)
        return {'bytes': values * (e + 1 + more * e) + 4 * scales + case['columns'] * e, 'flops': 8 * values}
    if not case['train']:
        return {'bytes': values * (2 + more) * e + case['columns'] * e, 'flops': 5 * values}
    # forward: x, residual in, y, residual out; backward: the residual stream, the gradients above, one below
    return {'bytes': values * (5 + (3 if more else 0)) * e + 3 * case['columns'] * e, 'flops': 16 * values}


# ---------------------------------------------------------------------------------------------------------
# the definitions in 64 bits: token after token, apart from the plain forms

def exact(case, seed):
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in prepare(case, seed).items()}
    with torch.no_grad():
        return {'scan': _exact_scan, 'scan_step': _exact_scan_step, 'conv': _exact_conv, 'conv_step': _exact_conv_step,
                'norm': _exact_norm, 'quantize': _exact_quantize}[case['op']](case, s)


def _exact_softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _silu_and_slope(x):
    sig = 1 / (1 + torch.exp(-x))
    return x * sig, sig * (1 + x * (1 - sig))


def _per_channel(x, case):
    """[batch, groups, states] -> [batch, channels, states]"""
    return x.repeat_interleave(case['channels'] // case['groups'], 1)


def _exact_scan(case, s):
    b, length, d, n = case['batch'], case['length'], case['channels'], case['states']
    ends = [length] * b if s['lengths'] is None else s['lengths'].tolist()
    live = torch.tensor([[t < e for e in ends] for t in range(length)], device='cuda')
    raw = s['delta'] + s['delta_bias']
    dt, (gate, slope) = _exact_softplus(raw), _silu_and_slope(s['z'])
    h, y = s['state'].clone(), torch.zeros_like(raw)
    kept = torch.empty(length + 1 if case['train'] else 0, b, d, n, dtype=torch.float64, device='cuda')
    if case['train']:
        kept[0] = h
    for t in range(length):
        on = live[t][:, None, None]
        new = torch.exp(dt[:, t, :, None] * s['A']) * h + (dt[:, t] * s['u'][:, t])[..., None] * _per_channel(s['B'][:, t], case)
        h = torch.where(on, new, h)
        y[:, t] = torch.where(on[..., 0], (h * _per_channel(s['C'][:, t], case)).sum(-1) + s['D'] * s['u'][:, t], 0.0)
        if case['train']:
            kept[t + 1] = h
    outs = [y * gate, h]
    if not case['train']:
        return outs
    on = live.t()[..., None]
    gout = torch.where(on, s['gout'], 0.0)
    gy, gz = gout * gate, gout * y * slope
    gu, gdt = torch.zeros_like(raw), torch.zeros_like(raw)
    gA, gB, gC = torch.zeros_like(s['A']), torch.zeros_like(s['B']), torch.zeros_like(s['C'])
    gh = s['gstate'].clone()
    by_group = (b, case['groups'], d // case['groups'], n)
    for t in reversed(range(length)):
        on_t = live[t][:, None, None]
        a = torch.exp(dt[:, t, :, None] * s['A'])
        now = gh + gy[:, t, :, None] * _per_channel(s['C'][:, t], case)
        now = torch.where(on_t, now, 0.0)
        q = now * a * kept[t]
        through = (now * _per_channel(s['B'][:, t], case)).sum(-1)
        gC[:, t] = (gy[:, t, :, None] * kept[t + 1]).view(by_group).sum(2)
        gB[:, t] = (now * (dt[:, t] * s['u'][:, t])[..., None]).view(by_group).sum(2)
        gA += (q * dt[:, t, :, None]).sum(0)
        gu[:, t] = through * dt[:, t] + s['D'] * gy[:, t]
        gdt[:, t] = (q * s['A']).sum(-1) + through * s['u'][:, t]
        gh = torch.where(on_t, a * now, gh)
    graw = gdt / (1 + torch.exp(-raw))
    return outs + [gu, graw, gA, gB, gC, (gy * s['u']).sum((0, 1)), gz, graw.sum((0, 1)), gh]


def _exact_scan_step(case, s):
    dt = _exact_softplus(s['delta'] + s['delta_bias'])
    h = torch.exp(dt[..., None] * s['A']) * s['state'] + (dt * s['u'])[..., None] * _per_channel(s['B'], case)
    y = (h * _per_channel(s['C'], case)).sum(-1) + s['D'] * s['u']
    return [y * _silu_and_slope(s['z'])[0], h]


def _exact_conv(case, s):
    b, length, taps = case['batch'], case['length'], case['taps']
    ends = [length] * b if s['lengths'] is None else s['lengths'].tolist()
    outs = [torch.zeros_like(s['x']), torch.zeros_like(s['state'])]
    grads = [torch.zeros_like(s[k]) for k in ('x', 'weight', 'bias', 'state')] if case['train'] else []
    for i, end in enumerate(ends):
        x = torch.cat([s['state'][i], s['x'][i, :end]])
        pre = s['bias'].expand(end, -1).clone()
        for k in range(taps):
            pre += s['weight'][:, k] * x[k:k + end]
        act, slope = _silu_and_slope(pre)
        outs[0][i, :end], outs[1][i] = act, x[end:]
        if case['train']:
            gpre = s['gout'][i, :end] * slope
            gx = torch.zeros_like(x)
            gx[end:] = s['gstate'][i]
            for k in range(taps):
                gx[k:k + end] += s['weight'][:, k] * gpre
                grads[1][:, k] += (gpre * x[k:k + end]).sum(0)
            grads[2] += gpre.sum(0)
            grads[3][i], grads[0][i, :end] = gx[:taps - 1], gx[taps - 1:]
    return outs + grads


def _exact_conv_step(case, s):
    x = torch.cat([s['state'], s['x'][:, None]], 1)
    pre = torch.einsum('bkd,dk->bd', x, s['weight']) + s['bias']
    return [_silu_and_slope(pre)[0], x[:, 1:]]


def _exact_normed(s):
    x = s['x'] if s['residual'] is None else s['x'] + s['residual']
    return x, 1 / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)


def _exact_norm(case, s):
    x, r = _exact_normed(s)
    outs = [x * r * s['weight']] + ([] if s['residual'] is None else [x])
    if not case['train']:
        return outs
    g = s['gout'] * s['weight']
    gx = r * g - x * r ** 3 * (g * x).sum(-1, keepdim=True) / x.shape[-1]
    if s['residual'] is not None:
        gx = gx + s['gres']
    return outs + [gx] * len(outs) + [(s['gout'] * x * r).sum(0)]


def _exact_quantize(case, s):
    x, r = _exact_normed(s)
    rows = x.shape[0]
    parts = (x * r * s['weight']).view(rows, -1, case['group'] or case['columns'])
    scale = torch.clamp(parts.abs().max(-1).values / 448, min=2.0 ** -126)
    v = parts / scale[..., None]
    # three bits behind the leading one, the smallest exponent -6: the nearest such value, ties to the even one
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))), min=-6) - 3)
    outs = [(torch.round(v / unit) * unit).clamp(-448, 448).view(rows, -1), scale]
    return outs if s['residual'] is None else outs + [x]
