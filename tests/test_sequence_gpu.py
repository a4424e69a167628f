"""The sequence operators on a device against their float64 statements (sequence_reference.py).

Tolerances.  An output of type t is the 32-bit result rounded once: at most eps(t) / 2 off, relatively.  The 32-bit result
of a recurrence over L tokens: a step multiplies the state's error by at most 1 + 2^-21 (the exponential and its rounded
argument: 2^-22; the multiply-adds: 2^-24 each) and adds terms rounded to 2^-24, so after L steps a sum of terms is off by
at most (L + 8) 2^-21 times the sum of the terms' magnitudes; sums over the states, channels or tokens behind it are sums of
such terms.  The magnitudes come from the same statement with the absolute values of all factors; where terms of both signs
meet that bounds their sum.  A backward pass runs two recurrences and an activation's derivative (at most 1.1): twice that.
"""
import pytest
import torch

import opveclib_b200 as ovl
import sequence_reference as ref
from helpers import DRYRUN

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(DRYRUN, reason='needs a device')]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEP32 = 2.0 ** -21


def _close(got, want, magnitude, steps):
    """|got - want| within half a step of got's type and (steps + 8) 2^-21 of the magnitudes."""
    want = want.detach().double()
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + (steps + 8) * STEP32 * magnitude + torch.finfo(got.dtype).tiny
    off = (got.detach().double() - want).abs()
    assert got.shape == want.shape
    # (a sum whose terms leave the range of 32 bits, or of got's type, has no value to be near to)
    off = torch.where(torch.as_tensor(magnitude < min(2.0 ** 120, torch.finfo(got.dtype).max), device=off.device), off, 0.0)
    assert bool((off <= bound).all()), 'off by %g, %g times the bound' % (off.max(), (off / bound).max())


def _normal(gen, *shape, scale=1.0, dtype=F32):
    return (torch.randn(shape, generator=gen, device='cuda') * scale).to(dtype)


def _generator(seed=0):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    return gen


def _top(x):
    return x.abs().amax() if x.numel() else 0.0


def _scan_case(t, batch, length, channels, states, groups=1, skip=True, gate=True, bias=True, softplus=True, initial=True,
               lengths=None, strided=False, seed=0):
    gen = _generator(seed)
    x = dict(u=_normal(gen, batch, length, channels, dtype=t),
             delta=_normal(gen, batch, length, channels, scale=0.5, dtype=t) if softplus
             else (0.01 + 0.2 * torch.rand(batch, length, channels, generator=gen, device='cuda')).to(t),
             A=-torch.rand(channels, states, generator=gen, device='cuda') * 4 - 0.1,
             B=_normal(gen, batch, length, groups, states, dtype=t), C=_normal(gen, batch, length, groups, states, dtype=t),
             D=_normal(gen, channels) if skip else None, z=_normal(gen, batch, length, channels, dtype=t) if gate else None,
             delta_bias=_normal(gen, channels, scale=0.3) - 3 if bias else None,
             initial_state=_normal(gen, batch, channels, states) if initial else None)
    if strided:                                                # halves of one projection, rows of another one with an odd width
        both = torch.cat([x['u'], x['z'] if gate else x['u']], -1)
        x['u'] = both[..., :channels]
        if gate:
            x['z'] = both[..., channels:]
        bc = torch.cat([x['B'].flatten(2), x['C'].flatten(2), x['C'].flatten(2)[..., :1]], -1)
        n = groups * states
        x['B'], x['C'] = bc[..., :n].unflatten(-1, (groups, states)), bc[..., n:2 * n].unflatten(-1, (groups, states))
        x['delta'] = x['delta'].transpose(0, 1).contiguous().transpose(0, 1)
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    return x, dict(delta_softplus=softplus, lengths=lengths)


def _doubles(x, grad=False, magnitude=False):
    out = {}
    for k, v in x.items():
        if v is not None:
            v = v.detach().double()
            v = v.abs() if magnitude and k not in ('A', 'delta', 'delta_bias') else v
            v = v.requires_grad_() if grad else v
        out[k] = v
    return out


def _check_scan(x, opts, backward=True, seed=1):
    length = x['u'].shape[1]
    gen = _generator(seed)
    want, want_h = ref.scan(**(xd := _doubles(x, grad=backward)), **opts)
    mag, mag_h = ref.scan(**(xm := _doubles(x, grad=backward, magnitude=True)), **opts, magnitude=True)
    xs = {k: v.detach().requires_grad_() if backward and v is not None else v for k, v in x.items()}
    out, h = ovl.selective_scan(**xs, **opts, return_state=True)
    assert out.dtype is x['u'].dtype and h.dtype is F32
    _close(out, want, mag.detach(), length)
    _close(h, want_h, mag_h.detach(), length)
    if not backward:
        return
    gout, gh = _normal(gen, *out.shape, dtype=out.dtype), _normal(gen, *h.shape)
    names = [k for k, v in x.items() if v is not None]
    got = torch.autograd.grad([out, h], [xs[k] for k in names], [gout, gh])
    wanted = torch.autograd.grad([want, want_h], [xd[k] for k in names], [gout.double(), gh.double()], allow_unused=True)
    mags = torch.autograd.grad([mag, mag_h], [xm[k] for k in names], [gout.double().abs(), gh.double().abs()], allow_unused=True)
    for k, g, w, m in zip(names, got, wanted, mags):
        assert g.dtype is x[k].dtype, k
        w = torch.zeros_like(g).double() if w is None else w
        m = torch.zeros_like(g).double() if m is None else m
        # (g(dt) adds a term through A < 0 to one through u B > 0: the sum of their magnitudes is bounded by the largest
        # of the tensor, not by the entry)
        m = m.abs() if k not in ('delta', 'delta_bias') else m.abs() + _top(m) + _top(w)
        try:
            _close(g, w, m, 2 * length)
        except AssertionError as e:
            raise AssertionError('gradient of %s: %s' % (k, e))


@pytest.mark.parametrize('t', [F32, F16, BF16])
@pytest.mark.parametrize('states', [1, 3, 4, 5, 16, 17, 32, 64, 65, 128])
def test_scan_states(t, states):
    _check_scan(*_scan_case(t, 2, 37, 24, states, groups=2))


@pytest.mark.parametrize('length', [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 100])
def test_scan_lengths(length):
    _check_scan(*_scan_case(BF16, 2, length, 40, 16))


@pytest.mark.parametrize('channels, groups', [(1, 1), (2, 2), (7, 1), (8, 1), (33, 1), (64, 1), (65, 1), (96, 3), (130, 2), (264, 4)])
def test_scan_channels_and_groups(channels, groups):
    _check_scan(*_scan_case(F32, 3, 19, channels, 16, groups=groups))


@pytest.mark.parametrize('left_out', ['skip', 'gate', 'bias', 'softplus', 'initial', 'all'])
@pytest.mark.parametrize('t', [F32, BF16])
def test_scan_without_optional_parts(t, left_out):
    names = ['skip', 'gate', 'bias', 'softplus', 'initial'] if left_out == 'all' else [left_out]
    _check_scan(*_scan_case(t, 2, 21, 40, 16, **{n: False for n in names}))


@pytest.mark.parametrize('t', [F32, F16, BF16])
def test_scan_without_softplus_keeps_steps_of_either_sign(t):
    x, opts = _scan_case(t, 2, 30, 40, 16, softplus=False, bias=False)
    x['delta_bias'] = torch.linspace(-0.005, 0.02, 40, device='cuda')          # some steps below zero: the state grows a little
    _check_scan(x, opts)


@pytest.mark.parametrize('t', [F32, BF16])
def test_scan_one_group_without_its_axis(t):
    x, opts = _scan_case(t, 2, 12, 16, 8)
    want = ovl.selective_scan(**x, **opts)
    x['B'], x['C'] = x['B'].squeeze(2), x['C'].squeeze(2)
    assert torch.equal(ovl.selective_scan(**x, **opts), want)


@pytest.mark.parametrize('t, channels, states', [(BF16, 64, 16), (BF16, 50, 16), (F32, 64, 5), (F16, 72, 24)])
def test_scan_strides(t, channels, states):
    _check_scan(*_scan_case(t, 3, 23, channels, states, strided=True))


@pytest.mark.parametrize('t', [F32, BF16])
def test_scan_takes_an_innermost_axis_that_is_not_contiguous_and_expanded_inputs(t):
    x, opts = _scan_case(t, 2, 12, 16, 8)
    want = ovl.selective_scan(**x, **opts)
    x['u'] = x['u'].transpose(1, 2).contiguous().transpose(1, 2)
    x['A'] = x['A'].t().contiguous().t()
    assert torch.equal(ovl.selective_scan(**x, **opts), want)
    x['z'] = x['z'][:1, :1].expand(2, 12, 16)                 # strides 0
    x['B'] = x['B'][:, :1].expand(2, 12, 1, 8)
    _check_scan(x, opts, backward=False)
    leaf = x['z'][:1, :1].detach().clone().requires_grad_()   # the gradient of a broadcast input is summed
    x['z'] = leaf.expand(2, 12, 16)
    out = ovl.selective_scan(**x, **opts)
    out.sum().backward()
    assert leaf.grad.shape == leaf.shape and bool(leaf.grad.abs().sum() > 0)


@pytest.mark.parametrize('t', [F32, BF16])
@pytest.mark.parametrize('lengths', [[0, 40, 17, 1], [16, 32, 39, 40], [0, 0, 0, 0], [-3, 41, 2 ** 31 - 1, 20]])
def test_scan_padding(t, lengths):
    x, opts = _scan_case(t, 4, 40, 48, 16, lengths=lengths)
    _check_scan(x, opts)
    out, h = ovl.selective_scan(**x, **opts, return_state=True)
    # whatever stands in the padding changes nothing, and no bit of a state that has seen no token
    for bad in (float('nan'), float('inf'), torch.finfo(t).min):
        y = {k: None if v is None else v.clone() for k, v in x.items()}
        for b, end in enumerate(lengths):
            end = max(0, min(end, 40))
            for k in ('u', 'delta', 'B', 'C', 'z'):
                y[k][b, end:] = bad
        for k, v in y.items():
            y[k] = v.requires_grad_()
        out2, h2 = ovl.selective_scan(**y, **opts, return_state=True)
        assert torch.equal(out2, out) and torch.equal(h2, h)
        gout = torch.full_like(out, bad)
        for b, end in enumerate(lengths):
            gout[b, :max(0, min(end, 40))] = 1
        grads = torch.autograd.grad(out2, list(y.values()), gout)
        for k, g in zip(y, grads):
            assert bool(torch.isfinite(g).all()), k
            if k in ('u', 'delta', 'B', 'C', 'z'):
                for b, end in enumerate(lengths):
                    assert not bool(g[b, max(0, min(end, 40)):].any()), k
    for b, end in enumerate(lengths):
        if end <= 0:
            assert torch.equal(h[b], x['initial_state'][b])
        assert not bool(out[b, max(0, min(end, 40)):].any())


@pytest.mark.parametrize('t, batch, length, channels, states, lengths', [
    (F32, 1, 700, 24, 16, None),                              # few channels: the length is cut into segments
    (BF16, 2, 515, 40, 16, [515, 130]), (F32, 1, 450, 8, 128, None), (BF16, 1, 400, 20, 4, None),
    (F32, 2, 333, 12, 64, [0, 260]),
])
def test_scan_segments(t, batch, length, channels, states, lengths):
    _check_scan(*_scan_case(t, batch, length, channels, states, lengths=lengths))


@pytest.mark.parametrize('t, batch, length, channels, states', [(BF16, 4, 18, 4096, 16), (F32, 8, 5, 2050, 16), (F16, 2, 9, 8192, 30)])
def test_scan_many_channels(t, batch, length, channels, states):
    _check_scan(*_scan_case(t, batch, length, channels, states))


def test_scan_bits_are_the_same_every_time_and_with_or_without_gradients():
    x, opts = _scan_case(BF16, 2, 300, 96, 16, lengths=[300, 111])
    xs = {k: v.requires_grad_() for k, v in x.items()}
    runs = []
    for _ in range(3):
        out, h = ovl.selective_scan(**xs, **opts, return_state=True)
        runs.append([out, h, *torch.autograd.grad([out, h], list(xs.values()), [torch.ones_like(out), torch.ones_like(h)])])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
    with torch.no_grad():
        out, h = ovl.selective_scan(**xs, **opts, return_state=True)
    assert torch.equal(out, runs[0][0]) and torch.equal(h, runs[0][1])


def test_scan_gradients_of_some_outputs_and_some_inputs():
    x, opts = _scan_case(F32, 2, 20, 16, 8)
    every = {k: v.clone().requires_grad_() for k, v in x.items()}
    out, h = ovl.selective_scan(**every, **opts, return_state=True)
    both = torch.autograd.grad(out.sum(), list(every.values()), retain_graph=True, allow_unused=True)
    only = torch.autograd.grad(h.sum(), [every['u'], every['initial_state']])
    assert bool(only[1].abs().sum() > 0)
    some = {k: v.clone().requires_grad_(k in ('A', 'z')) for k, v in x.items()}
    g = torch.autograd.grad(ovl.selective_scan(**some, **opts).sum(), [some['A'], some['z']])
    names = list(every)
    assert torch.equal(g[0], both[names.index('A')]) and torch.equal(g[1], both[names.index('z')])
    with pytest.raises(RuntimeError):                         # once differentiable
        first = torch.autograd.grad(ovl.selective_scan(**every, **opts).sum(), every['u'], create_graph=True)[0]
        first.sum().backward()


def test_scan_gradients_against_differences():
    """gradient . direction = (f(x + e v) - f(x - e v)) / 2e, with f in 64 bits: off by O(e^2) = 1e-8 relatively, below the
    32 bits of the gradient."""
    x, opts = _scan_case(F32, 2, 24, 16, 8, lengths=[24, 9])
    gen = _generator(5)
    w = _normal(gen, 2, 24, 16)
    xs = {k: v.clone().requires_grad_() for k, v in x.items()}
    grads = torch.autograd.grad((ovl.selective_scan(**xs, **opts) * w).sum(), list(xs.values()))
    for k, g in zip(xs, grads):
        v, e = _normal(gen, *x[k].shape).double(), 1e-4
        ends = []
        for sign in (1, -1):
            y = _doubles(x)
            y[k] = y[k] + sign * e * v
            ends.append((ref.scan(**y, **opts)[0] * w.double()).sum())
        slope, got = ((ends[0] - ends[1]) / (2 * e)).item(), (g.double() * v).sum().item()
        assert abs(slope - got) <= 2 * (48 + 8) * STEP32 * (g.double() * v).abs().sum().item() + 1e-6 * abs(slope) + 1e-6, k


@pytest.mark.parametrize('t', [F32, BF16])
def test_scan_in_pieces_is_the_scan(t):
    x, opts = _scan_case(t, 2, 64, 48, 16)
    out, h = ovl.selective_scan(**x, **opts, return_state=True)
    state, outs = x['initial_state'], []
    for a, b in ((0, 17), (17, 17), (17, 18), (18, 64)):
        part = {k: v[:, a:b] if k in ('u', 'delta', 'B', 'C', 'z') else v for k, v in x.items()}
        part['initial_state'] = state
        o, state = ovl.selective_scan(**part, **opts, return_state=True)
        outs.append(o)
    assert torch.equal(torch.cat(outs, 1), out) and torch.equal(state, h)   # the recurrence rounds every token alike


@pytest.mark.parametrize('t, rows, channels, states, groups', [
    (BF16, 1, 64, 16, 1), (BF16, 3, 40, 16, 2), (F32, 5, 7, 5, 1), (F16, 2, 130, 64, 2), (F32, 4, 9, 128, 3), (BF16, 2, 16, 1, 1),
    (BF16, 70, 4096, 16, 1), (F32, 66, 2500, 13, 4), (F16, 41, 1024, 128, 2), (BF16, 513, 512, 8, 1), (F32, 257, 4100, 3, 1),
])
def test_scan_step(t, rows, channels, states, groups):
    x, opts = _scan_case(t, rows, 1, channels, states, groups=groups)
    want, want_h = ref.scan(**_doubles(x), **opts)
    mag, mag_h = ref.scan(**_doubles(x, magnitude=True), **opts, magnitude=True)
    state = x.pop('initial_state').clone()
    step = {k: v[:, 0] if k in ('u', 'delta', 'B', 'C', 'z') else v for k, v in x.items()}
    out = ovl.selective_scan_step(state, **step, delta_softplus=True)
    assert out.dtype is t
    _close(out, want[:, 0], mag[:, 0], 1)
    _close(state, want_h, mag_h, 1)
    for name in ('D', 'z', 'delta_bias'):                     # left out one by one
        less = {**x, 'initial_state': state.clone()}
        less[name] = None
        want, want_h = ref.scan(**_doubles(less), delta_softplus=False)
        mag, mag_h = ref.scan(**_doubles(less, magnitude=True), delta_softplus=False, magnitude=True)
        if not bool(torch.isfinite(mag).all()):
            continue
        s = state.clone()
        out = ovl.selective_scan_step(s, **{**step, name: None})
        _close(out, want[:, 0], mag[:, 0] + 0.0, 8)
        _close(s, want_h, mag_h, 8)


@pytest.mark.parametrize('rows, channels', [(7, 40), (96, 4096)])
@pytest.mark.parametrize('op', ['scan', 'conv'])
def test_step_slots(op, rows, channels):
    """Rows with slots of their own anywhere in the cache; padding; a slot twice; one that does not exist.  What no row
    owns keeps its bits."""
    gen = _generator(3)
    n_slots = rows + 5
    slots = torch.randperm(n_slots, generator=gen, device='cuda')[:rows].to(torch.int32)
    slots[1], slots[3] = -1, slots[2].item()
    slots[4], slots[5] = n_slots, -2 ** 31
    good = [r for r in range(rows) if r not in (1, 3, 4, 5)]
    if op == 'scan':
        x, _ = _scan_case(BF16, rows, 1, channels, 16, initial=False)
        x.pop('initial_state')
        x = {k: v[:, 0] if k in ('u', 'delta', 'B', 'C', 'z') else v for k, v in x.items()}
        cache = _normal(gen, n_slots, channels, 16)

        def run(state, rows_of, slots=None):
            part = {k: v[rows_of] if k in ('u', 'delta', 'B', 'C', 'z') else v for k, v in x.items()}
            return ovl.selective_scan_step(state, **part, delta_softplus=True, slots=slots)
    else:
        x, w, b = _normal(gen, rows, channels, dtype=BF16), _normal(gen, channels, 4, dtype=BF16), _normal(gen, channels, dtype=BF16)
        cache = _normal(gen, n_slots, 3, channels, dtype=BF16)

        def run(state, rows_of, slots=None):
            return ovl.causal_conv1d_step(state, x[rows_of], w, b, 'silu', slots=slots)
    direct = cache[slots[good].long()].clone()
    want = run(direct, good)
    state = cache.clone()
    out = run(state, list(range(rows)), slots)
    assert torch.equal(out[good], want) and torch.equal(state[slots[good].long()], direct)
    untouched = torch.ones(n_slots, dtype=torch.bool, device='cuda')
    untouched[slots[good].long()] = False
    assert torch.equal(state[untouched], cache[untouched])
    assert not bool(out[[1, 5]].any()) and bool(out[[3, 4]].isnan().all())
    nothing = run(cache[:0].clone(), [0, 1], torch.tensor([0, -1], dtype=torch.int32, device='cuda'))
    assert bool(nothing[0].isnan().all()) and not bool(nothing[1].any())


# ---------------------------------------------------------------------------------------------------------
# convolution

def _conv_case(t, batch, length, channels, taps, bias=True, initial=True, params=None, seed=0):
    gen = _generator(seed)
    p = params or t
    return dict(x=_normal(gen, batch, length, channels, dtype=t), weight=_normal(gen, channels, taps, dtype=p),
                bias=_normal(gen, channels, dtype=p) if bias else None,
                initial_state=_normal(gen, batch, taps - 1, channels, dtype=t) if initial else None)


def _check_conv(x, activation, lengths=None, seed=1):
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    gen = _generator(seed)
    xd, xm = _doubles(x, grad=True), _doubles(x, grad=True, magnitude=True)
    want, want_s = ref.conv(**xd, activation=activation, lengths=lengths)
    mag, mag_s = ref.conv(**xm, activation=None, lengths=lengths)
    xs = {k: None if v is None else v.detach().requires_grad_() for k, v in x.items()}
    out, state = ovl.causal_conv1d(**xs, activation=activation, lengths=lengths, return_state=True)
    taps, tokens = x['weight'].shape[1], x['x'].shape[0] * x['x'].shape[1]
    # (silu doubles a relative error of its argument at most: |x silu'(x)| <= 2 |silu(x)| + ... <= 1.1 |x|)
    _close(out, want, 1.1 * mag.detach(), taps)
    assert torch.equal(state.double(), want_s)
    gout, gs = _normal(gen, *out.shape, dtype=out.dtype), _normal(gen, *state.shape, dtype=state.dtype)
    names = [k for k, v in x.items() if v is not None]
    got = torch.autograd.grad([out, state], [xs[k] for k in names], [gout, gs])
    wanted = torch.autograd.grad([want, want_s], [xd[k] for k in names], [gout.double(), gs.double()])
    mags = torch.autograd.grad([mag, mag_s], [xm[k] for k in names], [gout.double().abs(), gs.double().abs()])
    for k, g, w, m in zip(names, got, wanted, mags):
        assert g.dtype is x[k].dtype
        # an error of the argument reaches the derivative of silu with a factor of 0.5: relative to the largest sum
        slack = 0.5 * float(mag.detach().amax()) if mag.numel() else 0.0
        _close(g, w, m.abs() * (1.1 + slack), 4 * taps + min(tokens, 64) + tokens // 256)


@pytest.mark.parametrize('taps', [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize('t, activation', [(F32, None), (F16, 'silu'), (BF16, 'silu'), (BF16, None)])
def test_conv_taps(t, activation, taps):
    _check_conv(_conv_case(t, 2, 41, 40, taps), activation)


@pytest.mark.parametrize('length', [0, 1, 2, 3, 4, 7, 8, 31, 32, 33, 64, 65, 130, 300])
@pytest.mark.parametrize('taps', [4, 6])
def test_conv_lengths(length, taps):
    _check_conv(_conv_case(F32, 2, length, 24, taps), 'silu')


@pytest.mark.parametrize('channels', [1, 3, 7, 8, 12, 64, 129, 256, 260, 1024])
@pytest.mark.parametrize('t', [F32, BF16])
def test_conv_channels(t, channels):
    _check_conv(_conv_case(t, 2, 21, channels, 4), 'silu')


@pytest.mark.parametrize('bias, initial, params', [(False, True, None), (True, False, None), (False, False, F32), (True, True, F32)])
def test_conv_without_optional_parts_and_with_fp32_weights(bias, initial, params):
    _check_conv(_conv_case(BF16, 2, 40, 48, 4, bias, initial, params), 'silu')


@pytest.mark.parametrize('taps', [1, 3, 4, 8])
@pytest.mark.parametrize('lengths', [[0, 70, 17, 1], [2, 3, 69, 64], [0, 0, 0, 0], [-1, 71, 4, 5]])
def test_conv_padding(lengths, taps):
    x = _conv_case(BF16, 4, 70, 40, taps)
    _check_conv(x, 'silu', lengths)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    out, state = ovl.causal_conv1d(**x, activation='silu', lengths=n, return_state=True)
    for bad in (float('nan'), float('inf')):
        y = {k: v.clone() for k, v in x.items()}
        gout = torch.full_like(out, bad)
        for b, end in enumerate(lengths):
            y['x'][b, max(0, min(end, 70)):] = bad
            gout[b, :max(0, min(end, 70))] = 1
        y = {k: v.requires_grad_() for k, v in y.items()}
        out2, state2 = ovl.causal_conv1d(**y, activation='silu', lengths=n, return_state=True)
        assert torch.equal(out2, out) and torch.equal(state2, state)
        grads = torch.autograd.grad([out2, state2], list(y.values()), [gout, torch.zeros_like(state)])
        assert all(bool(torch.isfinite(g).all()) for g in grads)
        for b, end in enumerate(lengths):
            assert not bool(grads[0][b, max(0, min(end, 70)):].any())


@pytest.mark.parametrize('t, channels', [(BF16, 64), (BF16, 30), (F32, 64)])
def test_conv_strides(t, channels):
    x = _conv_case(t, 3, 50, channels, 4)
    want = ovl.causal_conv1d(**x, activation='silu')
    wide = torch.cat([x['x'], x['x']], -1)
    assert torch.equal(ovl.causal_conv1d(**{**x, 'x': wide[..., :channels]}, activation='silu'), want)
    assert torch.equal(ovl.causal_conv1d(**{**x, 'x': x['x'].transpose(0, 1).contiguous().transpose(0, 1)}, activation='silu'), want)
    assert torch.equal(ovl.causal_conv1d(**{**x, 'x': x['x'].transpose(1, 2).contiguous().transpose(1, 2)}, activation='silu'), want)
    _check_conv({**x, 'x': wide[..., channels:]}, 'silu')


@pytest.mark.parametrize('t, rows, channels, taps', [(BF16, 1, 64, 4), (F32, 3, 7, 2), (F16, 65, 300, 3), (BF16, 5, 33, 8), (F32, 2, 10, 1), (BF16, 200, 4096, 4)])
@pytest.mark.parametrize('activation', [None, 'silu'])
def test_conv_step_continues_the_convolution(t, rows, channels, taps, activation):
    x = _conv_case(t, rows, 12, channels, taps)
    want, want_s = ref.conv(**_doubles(x), activation=activation)
    mag, _ = ref.conv(**_doubles(x, magnitude=True))
    state = x['initial_state'].clone()
    for i in range(12):
        out = ovl.causal_conv1d_step(state, x['x'][:, i], x['weight'], x['bias'], activation)
        _close(out, want[:, i], 1.1 * mag[:, i], taps)
    assert torch.equal(state.double(), want_s)


# ---------------------------------------------------------------------------------------------------------
# norm

def _norm_case(t, rows, columns, residual=True, params=None, seed=0):
    gen = _generator(seed)
    return dict(x=_normal(gen, rows, columns, dtype=t), weight=(1 + 0.2 * _normal(gen, columns)).to(params or t),
                residual=_normal(gen, rows, columns, scale=2.0, dtype=t) if residual else None)


@pytest.mark.parametrize('columns', [1, 2, 7, 8, 100, 256, 257, 512, 1000, 1024, 1032, 2048, 2056, 4096, 5000, 8192, 16384, 16400, 32768])
@pytest.mark.parametrize('t', [F32, F16, BF16])
def test_norm_columns(t, columns):
    _check_norm(_norm_case(t, 5, columns))


@pytest.mark.parametrize('rows', [0, 1, 3, 4, 9, 700, 2000])
@pytest.mark.parametrize('residual, params', [(True, None), (False, F32)])
def test_norm_rows(rows, residual, params):
    _check_norm(_norm_case(BF16, rows, 264, residual, params))


def _check_norm(x, eps=1e-5, seed=1):
    gen = _generator(seed)
    xd = {k: None if v is None else v.detach().double().requires_grad_() for k, v in x.items()}
    want, want_s = ref.rms_norm(**xd, eps=eps)
    xs = {k: None if v is None else v.detach().requires_grad_() for k, v in x.items()}
    outs = ovl.rms_norm(**xs, eps=eps)
    outs = outs if x['residual'] is not None else (outs,)
    rows, columns = x['x'].shape
    # y: a dozen roundings and the sum of squares, which is off by at most its tree's depth + 8 terms in a row: < 64 steps
    # of 2^-24; the sum is exact to one rounding where both terms are of one sign, else relative to their magnitudes
    m_s = x['x'].double().abs() + (0 if x['residual'] is None else x['residual'].double().abs())
    r = 1 / torch.sqrt((want_s.detach() ** 2).mean(-1, keepdim=True) + eps)
    _close(outs[0], want, m_s * r * x['weight'].double().abs(), 0)
    if x['residual'] is not None:
        _close(outs[1], want_s, m_s * 2.0 ** -3, 0)
    above = [_normal(gen, *o.shape, dtype=o.dtype) for o in outs]
    names = [k for k, v in x.items() if v is not None]
    got = torch.autograd.grad(outs, [xs[k] for k in names], above)
    wanted = torch.autograd.grad([want, want_s][:len(outs)], [xd[k] for k in names], [g.double() for g in above])
    g = (above[0].double() * x['weight'].double()).abs()
    m_x = r * (g + m_s * r * (g * m_s * r).mean(-1, keepdim=True)) + (above[1].double().abs() if len(outs) > 1 else 0)
    mags = dict(x=m_x, residual=m_x, weight=(above[0].double().abs() * m_s * r).sum(0))
    for k, gg, w in zip(names, got, wanted):
        assert gg.dtype is x[k].dtype
        _close(gg, w, mags[k], 8 + (rows // 256 if k == 'weight' else 0))


def test_norm_shapes_strides_and_gradients_of_one_output():
    x = _norm_case(BF16, 12, 64)
    y, s = ovl.rms_norm(**x)
    y3, s3 = ovl.rms_norm(x['x'].view(3, 4, 64), x['weight'], x['residual'].view(3, 4, 64))
    assert torch.equal(y3.view(12, 64), y) and torch.equal(s3.view(12, 64), s) and y3.shape == (3, 4, 64)
    one = ovl.rms_norm(x['x'][0], x['weight'], x['residual'][0])
    assert torch.equal(one[0], y[0]) and one[0].shape == (64,)
    wide = torch.cat([x['x'], x['residual']], 1)
    ys, ss = ovl.rms_norm(wide[:, :64], x['weight'], wide[:, 64:])
    assert torch.equal(ys, y) and torch.equal(ss, s)
    odd = torch.cat([x['x'][:, :1], x['x'], x['residual']], 1)                  # rows of 129, off 16 bytes by one element
    yo, so = ovl.rms_norm(odd[:, 1:65], x['weight'], odd[:, 65:])
    assert torch.equal(so, s)
    torch.testing.assert_close(yo, y, rtol=2.0 ** -7, atol=0)                   # (another order of the sum: one step of bf16)
    yt, st = ovl.rms_norm(x['x'].t().contiguous().t(), x['weight'], x['residual'].expand(12, 64))
    assert torch.equal(yt, y) and torch.equal(st, s)
    leaves = [v.clone().requires_grad_() for v in x.values()]
    y, s = ovl.rms_norm(*[leaves[0], leaves[1], leaves[2]])
    gx, gr = torch.autograd.grad(s.sum(), [leaves[0], leaves[2]], retain_graph=True)
    assert torch.equal(gx, torch.ones_like(gx)) and torch.equal(gr, gx)
    gx, gr = torch.autograd.grad(y.sum(), [leaves[0], leaves[2]])
    assert torch.equal(gx, gr) and bool(gx.abs().sum() > 0)
    (y3, s3) = ovl.rms_norm(leaves[0], leaves[1], leaves[0])                    # x is its own residual: 2 x
    (y3.sum() + s3.sum()).backward()
    assert bool(torch.isfinite(leaves[0].grad).all())


@pytest.mark.parametrize('t', [F32, BF16])
@pytest.mark.parametrize('columns, group', [(8, None), (8, 8), (8, 1), (128, 128), (128, 64), (256, 32), (384, 128), (1000, 50), (1000, None),
                                            (1024, 256), (7, 7), (9, 3), (2048, None), (4096, 128), (4100, 4), (5120, 512), (16384, 128), (20000, None),
                                            (32768, 1)])
def test_norm_to_8_bits(t, columns, group):
    x = _norm_case(t, 6, columns, residual=columns % 3 != 0)
    got = ovl.rms_norm_quantize(**x, group=group)
    v, scale, s = ref.rms_norm_quantize(*[None if a is None else a.double() for a in x.values()], group=group)
    q, got_scale = got[0], got[1]
    assert q.dtype is torch.float8_e4m3fn and q.shape == x['x'].shape and got_scale.shape == scale.shape
    _close(got_scale, scale, scale, 8)
    # a value within the 32 bits' error of a border between two e4m3 values may go to either side
    near = (q.double() - v).abs() <= (ref.e4m3(v) - v).abs() * (1 + 1e-3) + 2.0 ** -17 * v.abs()
    assert bool(near.all())
    if x['residual'] is not None:
        assert torch.equal(got[2], ovl.rms_norm(**x)[1])
    else:
        assert len(got) == 2


def test_norm_to_8_bits_of_zeros_infinities_and_nan():
    x = torch.zeros(4, 256, device='cuda', dtype=BF16)
    x[1, 3], x[2, 200], x[3] = float('inf'), float('nan'), 1e-30
    w = torch.ones(256, device='cuda', dtype=BF16)
    q, scale = ovl.rms_norm_quantize(x, w, group=128, eps=0.0)
    assert bool(q[0].float().isnan().all())                    # 0 / 0: as the norm itself
    q, scale = ovl.rms_norm_quantize(x, w, group=128)
    assert not bool(q[0].float().any()) and bool((scale[0] == 2.0 ** -126).all())
    assert bool(q[1, 3].float().isnan()) and bool(scale[1, 0].isnan())
    assert bool(q[2].float().isnan().all()) and bool(scale[2].isnan().all())    # the row's mean square is NaN
    assert bool(torch.isfinite(q[3].float()).all())


# ---------------------------------------------------------------------------------------------------------
# together

class Block:
    """A state space block with random weights: norm, projections, convolution, scan, projection."""

    def __init__(self, t, width=64, channels=128, states=16, taps=4, seed=0):
        gen = _generator(seed)
        self.t, self.width, self.channels, self.states, self.taps = t, width, channels, states, taps
        self.norm = (1 + 0.1 * _normal(gen, width)).to(t)
        self.w_in, self.w_out = _normal(gen, width, 2 * channels, scale=width ** -0.5, dtype=t), _normal(gen, channels, width, scale=channels ** -0.5, dtype=t)
        self.w_x = _normal(gen, channels, channels + 2 * states, scale=channels ** -0.5, dtype=t)
        self.conv, self.conv_bias = _normal(gen, channels, taps, scale=0.5, dtype=t), _normal(gen, channels, scale=0.1, dtype=t)
        self.A, self.D = -torch.arange(1, states + 1, device='cuda').float().repeat(channels, 1), _normal(gen, channels)
        self.bias = _normal(gen, channels, scale=0.3) - 3

    def parameters(self):
        return [self.norm, self.w_in, self.w_out, self.w_x, self.conv, self.conv_bias, self.A, self.D, self.bias]

    def split(self, x):
        y = x @ self.w_x
        return y[..., :self.channels], y[..., self.channels:-self.states], y[..., -self.states:]

    def prompt(self, x, residual, conv_state, state, lengths=None):
        y, residual = ovl.rms_norm(x, self.norm, residual)
        y = y @ self.w_in
        u, conv_state = ovl.causal_conv1d(y[..., :self.channels], self.conv, self.conv_bias, 'silu', conv_state, lengths, True)
        delta, B, C = self.split(u)
        out, state = ovl.selective_scan(u, delta, self.A, B, C, self.D, y[..., self.channels:], self.bias, True, state, lengths, True)
        return out @ self.w_out, residual, conv_state, state

    def step(self, x, residual, conv_state, state, slots=None):
        y, residual = ovl.rms_norm(x, self.norm, residual)
        y = y @ self.w_in
        u = ovl.causal_conv1d_step(conv_state, y[:, :self.channels], self.conv, self.conv_bias, 'silu', slots)
        delta, B, C = self.split(u)
        out = ovl.selective_scan_step(state, u, delta, self.A, B, C, self.D, y[:, self.channels:], self.bias, True, slots)
        return out @ self.w_out, residual

    def plain(self, x, residual):
        w = [p.double() if not p.requires_grad else p for p in self.parameters()]
        norm, w_in, w_out, w_x, conv, conv_bias, A, D, bias = w
        y, s = ref.rms_norm(x, norm, residual)
        y = y @ w_in
        u, _ = ref.conv(y[..., :self.channels], conv, conv_bias, 'silu')
        d = u @ w_x
        out, _ = ref.scan(u, d[..., :self.channels], A, d[..., self.channels:-self.states], d[..., -self.states:], D,
                          y[..., self.channels:], bias, True)
        return out @ w_out, s


def test_block_answers_token_by_token_as_in_one_piece():
    block = Block(F32)
    gen = _generator(9)
    x, r = _normal(gen, 3, 20, 64), _normal(gen, 3, 20, 64)
    want, want_r = block.plain(x.double(), r.double())
    # a prompt of 12, 7 and 0 tokens, padded, then one token after the other in slots of a larger cache
    lengths = torch.tensor([12, 7, 0], dtype=torch.int32, device='cuda')
    zeros = torch.zeros(3, 3, 128, device='cuda'), torch.zeros(3, 128, 16, device='cuda')
    out, _, conv_state, state = block.prompt(x[:, :12].contiguous(), r[:, :12].contiguous(), *zeros, lengths)
    # matrix products in 32 bits (their own tolerance: 128 terms) around the operators: 1e-4 of the largest value
    top = want.abs().amax()
    for b, n in enumerate(lengths.tolist()):
        assert float((out[b, :n] - want[b, :n]).abs().amax() if n else 0) <= 1e-4 * top
    slots = torch.tensor([4, 1, 3], dtype=torch.int32, device='cuda')
    caches = torch.zeros(6, 3, 128, device='cuda'), torch.zeros(6, 128, 16, device='cuda')
    caches[0][slots.long()], caches[1][slots.long()] = conv_state, state
    at = lengths.long()
    rows = torch.arange(3, device='cuda')
    for _ in range(8):
        out, res = block.step(x[rows, at].contiguous(), r[rows, at].contiguous(), *caches, slots)
        assert float((out - want[rows, at]).abs().amax()) <= 1e-4 * top
        at = at + 1


def test_block_gradients():
    block = Block(F32)
    gen = _generator(11)
    x, r = _normal(gen, 2, 20, 64), _normal(gen, 2, 20, 64)
    zeros = torch.zeros(2, 3, 128, device='cuda'), torch.zeros(2, 128, 16, device='cuda')
    leaves = [x.requires_grad_(), r.requires_grad_()] + [p.requires_grad_() for p in block.parameters()]
    out, res, _, _ = block.prompt(x, r, *zeros)
    w, wr = _normal(gen, *out.shape), _normal(gen, *out.shape)
    got = torch.autograd.grad([out, res], leaves, [w, wr])
    doubles = [v.detach().double().requires_grad_() for v in leaves]
    other = Block(F32)
    (other.norm, other.w_in, other.w_out, other.w_x, other.conv, other.conv_bias, other.A, other.D, other.bias) = doubles[2:]
    out, res = other.plain(doubles[0], doubles[1])
    wanted = torch.autograd.grad([out, res], doubles, [w.double(), wr.double()])
    for g, want in zip(got, wanted):
        assert float((g - want).abs().amax()) <= 3e-4 * float(want.abs().amax())


def test_other_streams_and_captured_graphs():
    """A training step and a decoding step on a side stream, captured into two graphs and replayed in turn on new data."""
    block = Block(BF16)
    gen = _generator(13)
    data = [(_normal(gen, 2, 40, 64, dtype=BF16), _normal(gen, 2, 40, 64, dtype=BF16)) for _ in range(3)]
    zeros = torch.zeros(2, 3, 128, device='cuda', dtype=BF16), torch.zeros(2, 128, 16, device='cuda')
    leaves = [p.requires_grad_() for p in block.parameters()]

    def train(x, r):
        out, res, _, _ = block.prompt(x, r, *zeros)
        # (what is kept must not keep the eager graph: a leaf's accumulation node would tie a capture to its stream)
        return [out.detach(), *torch.autograd.grad([out, res], leaves, [torch.ones_like(out), torch.ones_like(res)])]

    def decode(x, caches):
        with torch.no_grad():
            return block.step(x, x, *caches)[0]

    eager = [[t.clone() for t in train(*d)] for d in data]
    fresh = lambda: (torch.zeros(2, 3, 128, device='cuda', dtype=BF16), torch.zeros(2, 128, 16, device='cuda'))  # noqa: E731
    caches = fresh()
    decoded = [decode(d[0][:, 0].contiguous(), caches) for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                             # another stream than the tensors' own
        for d, e in zip(data, eager):
            assert all(torch.equal(a, b) for a, b in zip(train(*d), e))
    torch.cuda.current_stream().wait_stream(side)
    sx, sr, st = data[0][0].clone(), data[0][1].clone(), data[0][0][:, 0].contiguous()
    caches = fresh()
    with torch.cuda.stream(side):
        train(sx, sr)
        decode(st, fresh())
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        captured = train(sx, sr)
    with torch.cuda.graph(g2):
        step = decode(st, caches)
    for c in caches:
        c.zero_()
    for d, e, s in zip(data, eager, decoded):
        sx.copy_(d[0]), sr.copy_(d[1]), st.copy_(d[0][:, 0])
        g2.replay()
        g1.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, e))
        assert torch.equal(step, s)


def test_a_state_changed_in_place_is_noticed_by_the_backward_pass():
    x, opts = _scan_case(F32, 2, 5, 16, 8)
    state = x['initial_state']
    x['u'] = x['u'].requires_grad_()
    out = ovl.selective_scan(**x, **opts)
    step = {k: v[:, 0].detach() if k in ('u', 'delta', 'B', 'C', 'z') else v for k, v in x.items() if k != 'initial_state'}
    ovl.selective_scan_step(state, **step)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()
    with torch.inference_mode():
        inside = torch.zeros(2, 16, 8, device='cuda')
        ovl.selective_scan_step(inside, **step)
        assert bool(inside.any())


def test_two_calls_at_once_on_two_streams():
    x, opts = _scan_case(BF16, 1, 600, 64, 16)                # cut into segments: both calls have workspaces
    want = ovl.selective_scan(**x, **opts, return_state=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ovl.selective_scan(**x, **opts, return_state=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason='needs two devices')
def test_tensors_on_another_device_than_the_current_one():
    x, opts = _scan_case(BF16, 1, 600, 64, 16)
    want = ovl.selective_scan(**x, **opts)
    other = {k: None if v is None else v.to('cuda:1') for k, v in x.items()}
    got = ovl.selective_scan(**other, **opts)
    assert got.device.index == 1 and torch.equal(got.cpu(), want.cpu())
    with pytest.raises(ValueError):
        ovl.selective_scan(**{**other, 'A': x['A']}, **opts)


def test_offsets_beyond_32_bits():
    """A strided input whose tokens lie more than 2^31 elements apart, and a cache of states larger than that."""
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip('needs 24 GB')
    x, opts = _scan_case(BF16, 1, 3, 64, 16)
    want = ovl.selective_scan(**x, **opts)
    far = torch.empty(3, (1 << 30) + 64, dtype=BF16, device='cuda')            # 2^30 + 64 elements per token
    u = far[None, :, 64:128]
    u.copy_(x['u'])
    assert u.stride(1) * 2 > 2 ** 31 and torch.equal(ovl.selective_scan(**{**x, 'u': u}, **opts), want)
    conv = _conv_case(BF16, 1, 3, 64, 4)
    want = ovl.causal_conv1d(**conv)
    u.copy_(conv['x'])
    assert torch.equal(ovl.causal_conv1d(**{**conv, 'x': u}), want)
    norm = _norm_case(BF16, 3, 64, residual=False)
    want = ovl.rms_norm(norm['x'], norm['weight'])
    u.copy_(norm['x'][None])
    assert torch.equal(ovl.rms_norm(u[0], norm['weight']), want)
    del far, u
    slots = (1 << 31) // (64 * 16) + 2
    cache = torch.zeros(slots, 64, 16, device='cuda')                          # 2^31 + 2048 states
    step = {k: v[:, 0] if k in ('u', 'delta', 'B', 'C', 'z') else v for k, v in x.items() if k != 'initial_state'}
    small = torch.zeros(1, 64, 16, device='cuda')
    want = ovl.selective_scan_step(small, **step, delta_softplus=True)
    at = torch.tensor([slots - 1], dtype=torch.int32, device='cuda')
    assert torch.equal(ovl.selective_scan_step(cache, **step, delta_softplus=True, slots=at), want)
    assert torch.equal(cache[-1], small[0]) and not bool(cache[0].any())


def test_empty_batches():
    x, opts = _scan_case(BF16, 0, 5, 16, 8)
    xs = {k: v.requires_grad_() for k, v in x.items()}
    out, h = ovl.selective_scan(**xs, **opts, return_state=True)
    assert out.shape == (0, 5, 16) and h.shape == (0, 16, 8)
    g = torch.autograd.grad(out.sum() + h.sum(), list(xs.values()))
    assert all(not bool(v.any()) for v in g)
    x = {k: v.requires_grad_() for k, v in _conv_case(BF16, 0, 5, 16, 4).items()}
    out = ovl.causal_conv1d(**x)
    assert all(not bool(v.any()) for v in torch.autograd.grad(out.sum(), [x['x'], x['weight'], x['bias']]))
    step = {k: v[:, 0] if k in ('u', 'delta', 'B', 'C', 'z') else v for k, v in xs.items() if k != 'initial_state'}
    with torch.no_grad():
        assert ovl.selective_scan_step(torch.zeros(0, 16, 8, device='cuda'), **step).shape == (0, 16)
    q, s = ovl.rms_norm_quantize(torch.zeros(0, 16, device='cuda'), torch.ones(16, device='cuda'))
    assert q.shape == (0, 16) and s.shape == (0, 1)


# ---- the compiled way of the usual calls --------------------------------------------------------------

from opveclib_b200 import sequence  # noqa: E402

def front_calls(dtype=torch.bfloat16):
    """name -> (call, the tensors it reads); every call draws the same inputs and returns a tuple."""
    g = torch.Generator().manual_seed(3)
    draw = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    u, z, dt = (draw(2, 21, 24).to(dtype).cuda() for _ in range(3))
    B, C = draw(2, 21, 2, 5).to(dtype).cuda(), draw(2, 21, 2, 5).to(dtype).cuda()
    A, D, h = -draw(24, 5).abs().cuda(), draw(24).cuda(), draw(2, 24, 5).cuda()
    w, bias, tail = draw(24, 4).cuda(), draw(24).cuda(), draw(2, 3, 24).to(dtype).cuda()
    lengths = torch.tensor([21, 9], dtype=torch.int32, device='cuda')
    slots = torch.tensor([1, 0], dtype=torch.int32, device='cuda')

    def step():
        state = h.clone()
        y = ovl.selective_scan_step(state, u[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], D, z[:, 0], D, True, slots)
        return y, state

    def conv_step():
        state = tail.clone()
        return ovl.causal_conv1d_step(state, u[:, 0], w, bias, 'silu', slots), state
    return {
        'scan': lambda: ovl.selective_scan(u, dt, A, B, C, D, z, D, True, h, lengths, True),
        'scan, least': lambda: (ovl.selective_scan(u, dt, A, B[:, :, 0], C[:, :, 0]),),
        'scan step': step,
        'conv': lambda: ovl.causal_conv1d(u, w, bias, 'silu', tail, lengths, True),
        'conv, least': lambda: (ovl.causal_conv1d(u, w.to(dtype)),),
        'conv step': conv_step,
        'norm': lambda: ovl.rms_norm(u, D, z),
        'norm, rows': lambda: (ovl.rms_norm(u[:, 0], D.to(dtype)),),
        'norm to 8 bits': lambda: ovl.rms_norm_quantize(u, D, z, 1e-5, 8),
        'norm to 8 bits, row': lambda: ovl.rms_norm_quantize(u[0], D),
    }


def bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


@pytest.mark.parametrize('name', [
    'scan', 'scan, least', 'scan step', 'conv', 'conv, least', 'conv step', 'norm', 'norm, rows', 'norm to 8 bits',
    'norm to 8 bits, row'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_the_compiled_way_is_taken_and_gives_the_same(name, dtype, monkeypatch):
    call = front_calls(dtype)[name]
    call()                                                   # (the first call loads it)
    assert sequence._front is not None
    taken = []
    monkeypatch.setattr(sequence, '_launch', lambda *a: taken.append(a))
    short = call()
    assert not taken                                         # nothing went through the long way
    monkeypatch.undo()
    monkeypatch.setattr(sequence, '_front', None)
    long = call()
    assert len(short) == len(long)
    for a, b in zip(short, long):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert torch.equal(bits(a), bits(b))


def test_the_compiled_way_leaves_alone_what_it_cannot_do():
    for call in front_calls().values():
        call()
    f = sequence._front
    x, w = torch.randn(4, 16, device='cuda'), torch.ones(16, device='cuda')
    assert f.rms_norm(x, w, None, 1e-6) is not None
    state, cx, cw = torch.zeros(4, 3, 16, device='cuda'), x, torch.ones(16, 4, device='cuda')
    assert f.causal_conv1d_step(state, cx, cw, None, None, None) is not None
    version = state._version
    for call in (lambda: f.rms_norm(x, w), lambda: f.rms_norm(x, w, None, 1), lambda: f.rms_norm(x.cpu(), w, None, 1e-6),
                 lambda: f.rms_norm(x, w.double(), None, 1e-6), lambda: f.rms_norm(x, w[:8], None, 1e-6),
                 lambda: f.rms_norm(x, w, x[:2], 1e-6), lambda: f.rms_norm(x.t(), w[:4], None, 1e-6),
                 lambda: f.rms_norm(x, w.clone().requires_grad_(), None, 1e-6, None),
                 lambda: f.rms_norm(x, w, None, -1e-6),
                 lambda: f.rms_norm(x, w, None, float('nan')), lambda: f.rms_norm(x, w, None, 1e-6, 3),
                 lambda: f.rms_norm(x, w, None, 1e-6, -1), lambda: f.rms_norm(x, w, None, 1e-6, 0),
                 lambda: f.rms_norm(x, w, None, 1e-6, True), lambda: f.rms_norm(x, w, None, 1e-6, 1 << 70),
                 lambda: f.rms_norm(torch._neg_view(x), w, None, 1e-6), lambda: f.rms_norm(None, w, None, 1e-6),
                 lambda: f.rms_norm(x.half(), w, x, 1e-6), lambda: f.rms_norm(x[0, 0], w, None, 1e-6),
                 lambda: f.causal_conv1d_step(state, cx, cw, None, 'tanh', None),
                 lambda: f.causal_conv1d_step(state[:2], cx, cw, None, None, None),
                 lambda: f.causal_conv1d_step(state[:, :2], cx, cw, None, None, None),
                 lambda: f.causal_conv1d_step(state, cx, cw, None, None, [0, 1, 2, 3])):
        assert call() is None
    assert state._version == version
    for bad in (dict(group=-1), dict(group=0), dict(group=True), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            ovl.rms_norm_quantize(x, w, **bad)


def test_views_of_negated_values():
    x, w = torch.randn(6, 32, device='cuda'), torch.ones(32, device='cuda')
    assert torch.equal(ovl.rms_norm(torch._neg_view(x), w), ovl.rms_norm(-x, w))
    taps = torch.randn(32, 4, device='cuda')
    assert torch.equal(ovl.causal_conv1d(x[None], torch._neg_view(taps)), ovl.causal_conv1d(x[None], -taps))


def test_forward_derivatives_are_refused():
    import torch.autograd.forward_ad as forward_ad
    x, w = torch.randn(6, 32, device='cuda'), torch.ones(32, device='cuda')
    ovl.rms_norm(x, w)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            ovl.rms_norm(dual, w)
        with pytest.raises(RuntimeError):
            ovl.rms_norm_quantize(dual, w)


def front_losses(dtype=torch.bfloat16):
    """name -> (call, names of the leaves it differentiates, the leaves): outputs of a call whose gradients are looked at."""
    g = torch.Generator().manual_seed(4)
    draw = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    seq = [draw(2, 37, 24).to(dtype) for _ in range(3)]
    bc = [draw(2, 37, 2, 5).to(dtype) for _ in range(2)]
    par = [-draw(24, 5).abs(), draw(24), draw(24), draw(2, 24, 5)]
    conv = [draw(24, 4), draw(24), draw(2, 3, 24).to(dtype)]
    lengths = torch.tensor([37, 18], dtype=torch.int32, device='cuda')
    return {
        'scan': (lambda u, dt, z, B, C, A, D, b, h: ovl.selective_scan(u, dt, A, B, C, D, z, b, True, h, lengths, True),
                 seq + bc + par),
        'scan, least': (lambda u, dt, B, C, A: (ovl.selective_scan(u, dt, A, B[:, :, 0], C[:, :, 1]),), seq[:2] + bc + par[:1]),
        'conv': (lambda x, w, b, h: ovl.causal_conv1d(x, w, b, 'silu', h, lengths, True), seq[:1] + conv),
        'conv, least': (lambda x, w: (ovl.causal_conv1d(x, w),), [seq[0], conv[0].to(dtype)]),
        'norm': (lambda x, r, w: ovl.rms_norm(x, w, r), seq[:2] + par[1:2]),
        'norm, rows': (lambda x, w: (ovl.rms_norm(x[:, 3], w),), [seq[0], par[1].to(dtype)]),
    }


@pytest.mark.parametrize('name', ['scan', 'scan, least', 'conv', 'conv, least', 'norm', 'norm, rows'])
@pytest.mark.parametrize('above', ['dense', 'broadcast', 'first only', 'last only'])
def test_gradients_of_the_compiled_way(name, above, monkeypatch):
    call, values = front_losses()[name]

    def gradients():
        leaves = [v.cuda().requires_grad_() for v in values]
        outs = list(call(*leaves))
        way = type(outs[0].grad_fn).__name__
        g = torch.Generator(device='cuda').manual_seed(5)
        top = [torch.randn(o.shape, generator=g, device='cuda').to(o.dtype) for o in outs]
        if above == 'broadcast':
            top = [t.flatten()[0].expand(o.shape) for t, o in zip(top, outs)]
        if above == 'first only':
            outs, top = outs[:1], top[:1]
        if above == 'last only':
            outs, top = outs[-1:], top[-1:]
        return way, torch.autograd.grad(outs, leaves, top)
    gradients()
    assert sequence._front is not None
    way, short = gradients()
    assert way not in ('SelectiveScanBackward', 'CausalConvBackward', 'RmsNormBackward')
    monkeypatch.setattr(sequence, '_front', None)
    way, long = gradients()
    assert way in ('SelectiveScanBackward', 'CausalConvBackward', 'RmsNormBackward')
    for a, b in zip(short, long):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize('front', [True, False])
@pytest.mark.parametrize('name', ['scan', 'conv', 'norm'])
def test_a_second_derivative_is_refused(name, front, monkeypatch):
    call, values = front_losses(torch.float32)[name]
    call(*(v.cuda() for v in values))
    if not front:
        monkeypatch.setattr(sequence, '_front', None)
    leaves = [v.cuda().requires_grad_() for v in values]
    loss = sum(o.sum() for o in call(*leaves))
    first = torch.autograd.grad(loss, leaves[0], create_graph=True)[0]      # the first derivative is there to be looked at
    assert bool(first.isfinite().all())
    with pytest.raises(RuntimeError, match='differentiable once'):
        (first ** 2).sum().backward()


def test_kept_tensors_changed_in_place_and_packed():
    call, values = front_losses()['norm, rows']
    call(*(v.cuda() for v in values))
    leaves = [v.cuda().requires_grad_() for v in values]
    x = leaves[0] * 2
    y, = call(x, leaves[1])
    x.mul_(2)
    with pytest.raises(RuntimeError, match='in-?place'):
        y.sum().backward()
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t.cpu(), lambda t: t.cuda()):
        y, = call(*leaves)
    y.sum().backward()
    assert packed and leaves[0].grad is not None
    y, = call(*leaves)
    y.sum().backward()
    with pytest.raises(RuntimeError, match='second time'):
        y.sum().backward()


@pytest.mark.parametrize('name', ['scan', 'conv', 'norm'])
@pytest.mark.parametrize('front', [True, False])
def test_checkpointed_calls(name, front, monkeypatch):
    """Checkpointing ends the repeated forward pass by an exception from where tensors are kept."""
    from torch.utils.checkpoint import checkpoint
    call, values = front_losses()[name]
    call(*(v.cuda() for v in values))
    if not front:
        monkeypatch.setattr(sequence, '_front', None)

    def gradients(run):
        leaves = [v.cuda().requires_grad_() for v in values]
        run(leaves).backward()
        return [v.grad for v in leaves]
    loss = lambda *leaves: sum(o.float().sum() for o in call(*leaves))  # noqa: E731
    want = gradients(lambda leaves: loss(*leaves))
    for reentrant in (False, True):
        got = gradients(lambda leaves: checkpoint(loss, *leaves, use_reentrant=reentrant))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('batch, length, channels, taps', [(2, 77, 1, 4), (3, 130, 31, 2), (1, 65, 257, 3), (2, 200, 519, 5)])
@pytest.mark.parametrize('skip', [0, 1])
def test_conv_rows_of_single_elements(dtype, batch, length, channels, taps, skip):
    """An odd number of 16-bit elements in a row, a first element in either half of a word: neighbours of other rows, and
    what stands in front of the tensor and behind it, are NaN."""
    gen = _generator(channels + skip)
    n = batch * length * channels
    memory = torch.full((n + 2 + skip,), float('nan'), device='cuda', dtype=dtype)
    x = memory[1 + skip:1 + skip + n].view(batch, length, channels)
    x.copy_(_normal(gen, batch, length, channels, dtype=dtype))
    w, b = _normal(gen, channels, taps, dtype=dtype), _normal(gen, channels, dtype=dtype)
    gout = _normal(gen, batch, length, channels + skip, dtype=dtype)[..., skip:]
    every = []
    for t in (x, x.float()):                                 # (rows of whole words: the other kernels)
        ts = [v.to(t.dtype).detach().requires_grad_() for v in (t, w, b)]
        if t is x:
            ts[0] = x.detach().requires_grad_()
        y = ovl.causal_conv1d(*ts, 'silu')
        every.append([y.detach(), *torch.autograd.grad(y, ts, gout.to(t.dtype))])
    for got, want in zip(*every):
        # one rounding of the same 32-bit sums (parameters' gradients: sums over tokens in another order, 2^-24 for each of
        # the terms, whose magnitudes are below 2^5)
        bound = torch.finfo(dtype).eps / 2 * want.abs() + batch * length * 2.0 ** -19 + torch.finfo(dtype).tiny
        assert bool(((got.float() - want).abs() <= bound).all())
