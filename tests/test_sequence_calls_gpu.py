"""Calls of the sequence operators that a program makes besides the plain ones: exact borders of the 8-bit output, gradients
that come from above as views of negated values, tracers, transforms and compilers around the calls."""
import pytest
import torch

import opveclib_b200 as ovl
import sequence_reference as ref
from opveclib_b200 import sequence
from helpers import DRYRUN

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(DRYRUN, reason='needs a device')]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---- the 8-bit output is a quotient ------------------------------------------------------------------------------

@pytest.mark.parametrize('columns, group', [(8, 8), (128, None), (1024, 256), (2048, None), (4096, 128), (4096, 16), (8192, 512),
                                            (4096, 4), (512, 2), (1000, 50), (1000, None), (4100, 4), (32768, 32)])
@pytest.mark.parametrize('size', [1.0, 2.0 ** -128, 2.0 ** -119, 2.0 ** -40, 2.0 ** 118])
@pytest.mark.parametrize('t', [F32, BF16])
def test_norm_to_8_bits_next_to_the_borders(t, columns, group, size):
    """Rows of +1 and -1 have the mean square 1, so y is the weight exactly, and scale and q follow from the weight without
    any other rounding than those of the two quotients and of the e4m3 value: equal, not near.  The weights are the borders
    between e4m3 values times the scale, up to three steps of 32 bits to either side."""
    gen = torch.Generator().manual_seed(columns + (group or 0))
    n = group or columns
    top = (1 + torch.rand(columns // n, generator=gen)) * 448 * size
    top[0] = (2 - 2.0 ** -23) * 448 * size                                      # a scale whose fraction is all ones, or next to it
    scale = torch.clamp(top / 448, min=2.0 ** -126)                             # (on the CPU: rounded correctly)
    borders = torch.cat([torch.tensor([(1 + (2 * i + 1) / 16) * 2.0 ** e for e in range(-6, 9) for i in range(8)][:-2]),
                         torch.tensor([(2 * i + 1) * 2.0 ** -10 for i in range(8)])])
    w = borders[torch.randint(len(borders), (columns // n, n), generator=gen)] * scale[:, None]
    away = torch.randint(-3, 4, w.shape, generator=gen)
    w = (w.view(torch.int32) + away.to(torch.int32)).view(F32)
    w = torch.minimum(w, top[:, None])
    w[:, 0] = top
    want = (w / scale[:, None]).to(torch.float8_e4m3fn).flatten()
    w = w.flatten().cuda()
    x = torch.where(torch.rand(3, columns, generator=gen) < 0.5, -1.0, 1.0).to(t).cuda()
    assert torch.equal(ovl.rms_norm(x.float(), w, eps=0.0), x.float() * w)      # what the test stands on
    q, got_scale = ovl.rms_norm_quantize(x, w, eps=0.0, group=group)
    for row in range(3):
        assert torch.equal(got_scale[row].cpu(), scale)
        assert torch.equal(q[row].cpu().float(), want.float() * x[row].cpu().float())


def test_norm_to_8_bits_of_an_infinite_weight():
    """Its group has an infinite scale: the finite values are zeros, the infinite one NaN; the other groups are as ever."""
    x = torch.ones(2, 256, device='cuda')
    w = torch.ones(256, device='cuda')
    w[5] = float('inf')
    for group, inside in ((128, 128), (None, 256), (64, 64), (2, 2)):
        q, scale = ovl.rms_norm_quantize(x, w, eps=0.0, group=group)
        at = 5 // inside
        assert bool(torch.isinf(scale[:, at]).all()) and int(torch.isinf(scale).sum()) == 2
        assert bool(q[:, 5].float().isnan().all())
        mine = q[:, at * inside:(at + 1) * inside].float()
        assert int(mine.isnan().sum()) == 2 and not bool(torch.nan_to_num(mine).any())
        assert bool((q[:, (at + 1) * inside:].float() == 448).all())


# ---- gradients from above that are views of negated values -------------------------------------------------------

def losses(t=F32):
    """name -> (call that returns all outputs, its leaves)"""
    gen = torch.Generator().manual_seed(11)
    draw = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    seq, bc = [draw(2, 9, 8).to(t) for _ in range(3)], [draw(2, 9, 2, 4).to(t) for _ in range(2)]
    par, conv = [-draw(8, 4).abs(), draw(8), draw(8), draw(2, 8, 4)], [draw(8, 4), draw(8), draw(2, 3, 8).to(t)]
    return {
        'scan': (lambda u, dt, z, B, C, A, D, b, h: ovl.selective_scan(u, dt, A, B, C, D, z, b, True, h, None, True), seq + bc + par),
        'conv': (lambda x, w, b, h: ovl.causal_conv1d(x, w, b, 'silu', h, None, True), seq[:1] + conv),
        'norm': (lambda x, r, w: ovl.rms_norm(x, w, r), seq[:2] + par[1:2]),
        'norm, rows': (lambda x, r, w: ovl.rms_norm(x[:, 0], w, r[:, 0]), seq[:2] + par[1:2]),
    }


@pytest.mark.parametrize('front', [True, False])
@pytest.mark.parametrize('which', [(0,), (1,), (0, 1)])
@pytest.mark.parametrize('name', ['scan', 'conv', 'norm', 'norm, rows'])
@pytest.mark.parametrize('t', [F32, BF16])
def test_gradients_from_above_that_are_negated_views(t, name, which, front, monkeypatch):
    call, values = losses(t)[name]
    call(*(v.cuda() for v in values))                         # (the first call loads the compiled way)
    if front:
        assert sequence._front is not None
    else:
        monkeypatch.setattr(sequence, '_front', None)
    leaves = [v.cuda().requires_grad_() for v in values]
    outs = call(*leaves)
    gen = torch.Generator(device='cuda').manual_seed(12)
    above = [torch.randn(o.shape, generator=gen, device='cuda').to(o.dtype) for o in outs]

    def grads(views):
        pick = [outs[i] for i in which]
        top = [torch._neg_view(-above[i]) if views else above[i] for i in which]
        assert all(g.is_neg() == views for g in top)
        return torch.autograd.grad(pick, leaves, top, retain_graph=True, allow_unused=True)
    for got, want in zip(grads(True), grads(False)):
        assert (got is None) == (want is None)
        assert got is None or torch.equal(got, want)


@pytest.mark.parametrize('front', [True, False])
def test_a_gradient_through_a_conjugated_complex_number(front, monkeypatch):
    """One channel, and an output that becomes the imaginary part of a number whose conjugate is used further on: the
    gradient comes back as a view of negated values with the stride 1 at its end."""
    gen = torch.Generator(device='cuda').manual_seed(13)
    draw = lambda *shape: torch.randn(*shape, generator=gen, device='cuda')  # noqa: E731
    w, a, factor = draw(1, 3), draw(2, 5), torch.complex(draw(2, 5), draw(2, 5))
    x = draw(2, 5, 1)
    ovl.causal_conv1d(x, w)
    if not front:
        monkeypatch.setattr(sequence, '_front', None)

    def gradient(conv, x, a, factor):
        x = x.detach().requires_grad_()
        (torch.complex(a, conv(x).squeeze(-1)).conj() * factor).real.sum().backward()
        return x.grad
    got = gradient(lambda v: ovl.causal_conv1d(v, w, activation='silu'), x, a, factor)
    want = gradient(lambda v: ref.conv(v, w.double(), activation='silu')[0], x.double(), a.double(), factor.to(torch.complex128))
    # sums of three products with silu's derivative (at most 1.1), 32 bits throughout: 16 roundings of at most 2^-24
    assert bool(((got.double() - want).abs() <= 2.0 ** -20 * 1.1 * 3 * w.abs().max() * factor.abs().max()).all())


# ---- tracers ------------------------------------------------------------------------------------------------------

def plain_calls():
    """name -> (call of one tensor, the tensor)"""
    gen = torch.Generator().manual_seed(14)
    draw = lambda *shape: torch.randn(*shape, generator=gen).cuda()  # noqa: E731
    x, w, taps, A, B = draw(2, 6, 8), draw(8), draw(8, 4), -draw(8, 4).abs(), draw(2, 6, 4)
    state, tail = draw(2, 8, 4), draw(2, 3, 8)
    return {
        'scan': (lambda v: ovl.selective_scan(v, v, A, B, B, delta_softplus=True), x),
        'conv': (lambda v: ovl.causal_conv1d(v, taps), x),
        'norm': (lambda v: ovl.rms_norm(v, w), x),
        'norm to 8 bits': (lambda v: ovl.rms_norm_quantize(v, w)[1], x),
        'scan step': (lambda v: ovl.selective_scan_step(state, v, v, A, B[:, 0], B[:, 0], delta_softplus=True), x[:, 0]),
        'conv step': (lambda v: ovl.causal_conv1d_step(tail, v, taps), x[:, 0]),
    }


NAMES = ['scan', 'conv', 'norm', 'norm to 8 bits', 'scan step', 'conv step']


@pytest.mark.parametrize('front', [True, False])
@pytest.mark.parametrize('name', NAMES)
@pytest.mark.parametrize('tracer', ['jit', 'fx', 'fx before dispatch'])
def test_tracing_is_refused(tracer, name, front, monkeypatch):
    """A trace would keep the example's answer."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, x = plain_calls()[name]
    call(x)
    if not front:
        monkeypatch.setattr(sequence, '_front', None)
    with torch.no_grad(), pytest.raises(RuntimeError, match='cannot be traced'):
        if tracer == 'jit':
            torch.jit.trace(lambda v: call(v * 2), (x,), check_trace=False)
        else:
            make_fx(lambda v: call(v * 2), pre_dispatch=tracer != 'fx')(x)
    call(x)                                                   # and is over with the tracer


# ---- tensors without memory of their own --------------------------------------------------------------------------

@pytest.mark.parametrize('front', [True, False])
def test_a_tensor_without_memory_does_not_count_as_left_out(front, monkeypatch):
    """torch.func.functionalize hands over tensors whose address is null; where a tensor may be left out, null means that."""
    x, r, w = torch.randn(4, 16, device='cuda'), torch.randn(4, 16, device='cuda'), torch.ones(16, device='cuda')
    taps, b = torch.randn(16, 4, device='cuda'), torch.randn(16, device='cuda')
    ovl.rms_norm(x, w, r)
    if not front:
        monkeypatch.setattr(sequence, '_front', None)
    for call, v in ((lambda v: ovl.rms_norm(x, w, v)[0], r), (lambda v: ovl.causal_conv1d(x[None], taps, v), b),
                    (lambda v: ovl.rms_norm(v, w), x), (lambda v: ovl.rms_norm_quantize(x, w, v)[1], r)):
        with pytest.raises(RuntimeError):
            torch.func.functionalize(call)(v)


# ---- what the documents say of transforms and compilers -----------------------------------------------------------

@pytest.mark.parametrize('front', [True, False])
@pytest.mark.parametrize('name', NAMES)
def test_transforms_are_refused(name, front, monkeypatch):
    call, x = plain_calls()[name]
    call(x)
    if not front:
        monkeypatch.setattr(sequence, '_front', None)
    total = lambda v: call(v).float().sum()  # noqa: E731
    for transform in (lambda: torch.func.grad(total)(x), lambda: torch.func.vmap(call)(x[None].expand(2, *x.shape)),
                      lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.jacrev(call)(x),
                      lambda: torch.func.functionalize(call)(x)):
        with pytest.raises(RuntimeError):
            transform()


@pytest.mark.parametrize('front', [True, False])
@pytest.mark.parametrize('name', ['scan', 'conv', 'norm'])
def test_batched_gradients_are_refused(name, front, monkeypatch):
    call, x = plain_calls()[name]
    call(x)
    if not front:
        monkeypatch.setattr(sequence, '_front', None)
    leaf = x.clone().requires_grad_()
    out = call(leaf)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaf, torch.ones(3, *out.shape, device='cuda'), is_grads_batched=True)


@pytest.mark.parametrize('front', [True, False])
@pytest.mark.parametrize('name', NAMES)
@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_a_compiler_runs_the_operators_between_its_graphs(backend, name, front, monkeypatch):
    call, x = plain_calls()[name]
    call(x)
    if not front:
        monkeypatch.setattr(sequence, '_front', None)
    torch._dynamo.reset()
    compiled = torch.compile(lambda v: call(v * 2) + 1, backend=backend)
    for k in range(3):
        call, x = plain_calls()[name]                         # (steps change their state: the same one for both)
        with torch.no_grad():
            want = call((x + k) * 2) + 1
        call, x = plain_calls()[name]
        with torch.no_grad():
            assert torch.equal(compiled(x + k), want)
    if 'step' in name or name == 'norm to 8 bits':
        return
    leaf, other = x.clone().requires_grad_(), x.clone().requires_grad_()
    torch.autograd.backward((call(leaf * 2) + 1).sum())
    torch.autograd.backward(torch.compile(lambda v: call(v * 2) + 1, backend=backend)(other).sum())
    assert torch.equal(leaf.grad, other.grad)
    with pytest.raises(Exception):                            # (whatever the compiler raises)
        torch.compile(lambda v: call(v * 2) + 1, backend=backend, fullgraph=True)(x)


# ---- many states ---------------------------------------------------------------------------------------------------

def test_scan_gradients_with_the_parts_of_gB_and_gC_in_several_pieces():
    """4096 channels of 128 states: the channel tiles' parts of gB and gC do not fit the work space at once.  Quarters of the
    channels are calls without pieces.  Gradients that a channel has for itself are the same bits; gB and gC are the
    quarters' sum, and as all terms are positive here, two sums of the same 1024 tiles' parts in different orders differ by
    at most 2 x 1024 roundings of 2^-24."""
    gen = torch.Generator(device='cuda').manual_seed(15)
    batch, length, channels, states = 1, 2048, 4096, 128
    draw = lambda *shape: torch.rand(*shape, generator=gen, device='cuda') + 0.1  # noqa: E731
    u, delta, gout = draw(batch, length, channels), draw(batch, length, channels) - 3, draw(batch, length, channels)
    B, C, A = draw(batch, length, states), draw(batch, length, states), -4 * draw(channels, states)
    lengths = torch.tensor([length - 37], dtype=torch.int32, device='cuda')

    def grads(part):
        leaves = [v.clone().requires_grad_() for v in (u[..., part], delta[..., part], A[part], B, C)]
        out = ovl.selective_scan(*leaves, delta_softplus=True, lengths=lengths)
        return torch.autograd.grad(out, leaves, gout[..., part])
    every, again = grads(slice(0, channels)), grads(slice(0, channels))
    assert all(torch.equal(a, b) for a, b in zip(every, again))
    quarters = [grads(slice(k * channels // 4, (k + 1) * channels // 4)) for k in range(4)]
    for i, axis in ((0, -1), (1, -1), (2, 0)):
        assert torch.equal(every[i], torch.cat([q[i] for q in quarters], axis))
    for i in (3, 4):
        want = sum(q[i].double() for q in quarters)
        assert bool((want[:, :length - 37] > 0).all()) and not bool(every[i][:, length - 37:].any())
        assert bool(((every[i].double() - want).abs() <= 2.0 ** -13 * want).all())
