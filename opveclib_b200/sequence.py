"""Operators on sequences: the parts of a state space block between its matrix products, as hand-written kernels.

``selective_scan``   the recurrence ``h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t``, ``y_t = C_t . h_t + D u_t``, optionally
                     gated by ``silu(z_t)``: an accumulation whose factor depends on the data, which the operator
                     language's ``accumulate`` (opveclib/examples/test_accumulate.py:22-78) cannot express in parallel
``causal_conv1d``    the short convolution in front of it, every channel by itself (the reference's ``conv_1d``,
                     opveclib/examples/conv1D.py:18-203, sums over all channels)
``rms_norm``         the root-mean-square norm with the residual's addition; ``rms_norm_quantize`` writes 8 bits and scales
``selective_scan_step``, ``causal_conv1d_step``   one token for each of many sequences, their states updated in place

All take torch CUDA tensors of one type (float32, float16 or bfloat16), compute in 32 bits and round once.  Kernels run
on torch's current stream of the tensors' device through the C-ABI library (``include/ovl_b200.h``); workspaces come from
torch's allocator on that stream, so calls can be captured into CUDA graphs.  The first three are differentiable (once;
every gradient is computed, also those of inputs that need none).
A tensor whose innermost axis is not contiguous is copied first, any other strides are taken as they are.  Wrong types
raise ``TypeError``, wrong shapes and values ``ValueError``, before anything is launched; tracers (``torch.jit.trace``,
``torch.export``) and the transforms of ``torch.func`` are refused with a ``RuntimeError``.
"""
import struct

from . import launcher
from .local import logger

_torch_module = None
#: the compiled short way of the usual calls (csrc/ovl_front.cpp), once the library is loaded
_front = None
_front_tried = False
_codes = None
_raw_stream = None
_current_device = None
_forward_ad = None
_entries = {}


def _torch():
    global _torch_module, _codes, _raw_stream, _current_device, _forward_ad
    if _torch_module is None:
        import torch
        _codes = {torch.float16: 1, torch.float32: 2, torch.bfloat16: 12}
        # the current stream's handle without the Stream object around it (2 us of a small call)
        _raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)
        if _raw_stream is None:
            _raw_stream = lambda index: torch.cuda.current_stream(index).cuda_stream  # noqa: E731
        # (asked for only once tensors are known to be CUDA tensors: the runtime is up then)
        _current_device = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)
        from torch.autograd import forward_ad
        _forward_ad = forward_ad
        _torch_module = torch
    return _torch_module


_TWO = struct.Struct('2q')
_SCAN = struct.Struct('47q')
_SCAN_STEP = struct.Struct('25q')
_CONV = struct.Struct('26q')
_CONV_STEP = struct.Struct('14q')
_NORM = struct.Struct('5qd17q')
#: most states of a scan's channel, taps of a convolution, columns of a norm's row
MAX_STATES, MAX_TAPS, MAX_COLUMNS = 128, 8, 32768


def _ptr(x):
    """The address of what may be left out (0): a tensor has one unless it is empty (those of torch.func.functionalize and of
    other wrappers do not, and would count as left out)."""
    if x is None:
        return 0
    address = x.data_ptr()
    if not address and x.numel():
        raise RuntimeError('opveclib_b200 needs tensors with memory of their own, not %s' % type(x).__name__)
    return address


def _refuse(x, name, shape, dtype, what):
    if not isinstance(x, _torch_module.Tensor):
        raise TypeError('%s: %s must be a torch tensor' % (what, name))
    if x.dtype is not dtype:
        raise TypeError('%s: %s must be %s, not %s' % (what, name, dtype, x.dtype))
    raise ValueError('%s: %s must have the shape %s, not %s' % (what, name, tuple(shape), tuple(x.shape)))


def _tensor(x, name, shape, dtype, what):
    """Refuse anything but a tensor of this shape and type; a copy where the innermost axis is not contiguous."""
    try:
        right = x.dtype is dtype and x.shape == shape
    except AttributeError:
        right = False
    if not right:
        _refuse(x, name, shape, dtype, what)
    if x.is_neg():
        x = x.resolve_neg()
    return x if x.is_contiguous() or x.stride(-1) == 1 else x.contiguous()


def _dense(x, name, shape, dtype, what):
    try:
        right = x.dtype is dtype and x.shape == shape
    except AttributeError:
        right = False
    if not right:
        _refuse(x, name, shape, dtype, what)
    if x.is_neg():
        x = x.resolve_neg()
    return x if x.is_contiguous() else x.contiguous()


def _refuse_tracers(what):
    """The kernels are launched past torch's dispatcher: a tracer would keep this call's answer, or memory that nothing
    fills, and miss the states changed in place.  (torch.jit.trace; torch.fx's tracer of real tensors, before or behind
    dispatch; torch.export on top of it.)"""
    torch = _torch_module
    if torch.jit.is_tracing() or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None \
            or torch._ops._len_torch_dispatch_stack_pre_dispatch() > 0:
        raise RuntimeError('%s cannot be traced: call it outside of the trace' % what)


def _first(x, name, rank, what):
    torch = _torch()
    _refuse_tracers(what)
    if not isinstance(x, torch.Tensor):
        raise TypeError('%s: %s must be a torch tensor' % (what, name))
    if x.dtype not in _codes:
        raise TypeError('%s: %s must be float32, float16 or bfloat16, not %s' % (what, name, x.dtype))
    if rank is not None and x.dim() != rank:
        raise ValueError('%s: %s must have %d axes, not %d' % (what, name, rank, x.dim()))
    return torch


def _state(x, name, rank, dtype, what):
    """A state that is updated in place has to be dense: a copy would be updated instead of it."""
    if not isinstance(x, _torch_module.Tensor):
        raise TypeError('%s: %s must be a torch tensor' % (what, name))
    if x.dtype is not dtype:
        raise TypeError('%s: %s must be %s, not %s' % (what, name, dtype, x.dtype))
    if x.dim() != rank:
        raise ValueError('%s: %s must have %d axes, not %d' % (what, name, rank, x.dim()))
    if not x.is_contiguous() or x.is_neg():
        raise ValueError('%s: %s is updated in place and must be contiguous' % (what, name))


def _index(x, name, n, what):
    if x is None:
        return None
    return _dense(x, name, (n,), _torch_module.int32, what)


def _one_device(what, *tensors):
    device = tensors[0].device
    if device.type != 'cuda':
        raise RuntimeError('%s: opveclib_b200 needs CUDA tensors: there is no CPU execution path' % what)
    for x in tensors:
        if x is not None and x.device != device:
            raise ValueError('%s: all tensors must be on one device, found %s and %s' % (what, device, x.device))
    return device


#: what ovl_front.cpp calls, in the order of its bind()
_FRONT_ENTRIES = ('ovl_selective_scan', 'ovl_selective_scan_backward', 'ovl_selective_scan_step', 'ovl_causal_conv',
                  'ovl_causal_conv_backward', 'ovl_causal_conv_step', 'ovl_rms_norm', 'ovl_rms_norm_backward',
                  'ovl_selective_scan_workspace_bytes', 'ovl_causal_conv_workspace_bytes', 'ovl_rms_norm_workspace_bytes')


def _load_front():
    """From the second call on the usual ones take the compiled way from their arguments to the launch.  Measured, call by
    call: scan, one token for one sequence, 14.7 -> 5.2 us; convolution, one token for 64, 11.7 -> 5.2; a norm of 8 rows to
    8 bits 17 -> 6.4; forward and backward of a convolution whose kernels take 20 us, 117 -> 63.  The same kernels run
    without it: where it cannot be built, that is logged and no more."""
    global _front, _front_tried
    _front_tried = True
    import ctypes
    import importlib.util
    from . import compiler
    try:
        path = compiler.build_front()
        if path is None:
            raise ImportError('no C++ compiler')
        spec = importlib.util.spec_from_file_location('ovl_front', path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        library = launcher.library()
        module.bind(_torch().nn.Parameter,
                    *(ctypes.cast(getattr(library, name), ctypes.c_void_p).value for name in _FRONT_ENTRIES))
    except (ImportError, OSError, RuntimeError) as e:
        logger.warning('the compiled way of the sequence operators\' calls is not used: %s', e)
    else:
        _front = module


def _launch(name, args, device):
    """Enqueue on torch's current stream of the tensors' device, whichever device is the current one."""
    function = _entries.get(name)
    if function is None:
        function = _entries[name] = getattr(launcher.library(), name)
        if not _front_tried:
            _load_front()
    index = device.index
    if index == _current_device():
        status = function(args, _raw_stream(index))
    else:
        with _torch_module.cuda.device(device):
            status = function(args, _raw_stream(index))
    if status:
        launcher.check(status, name)


def _with_workspace(args, at, size, x):
    """The packed arguments with a workspace of ``size`` bytes, on the device of ``x``, in the fields ``at`` and ``at + 1``,
    and the workspace, which the caller holds until the launch."""
    if not size:
        return args, None
    workspace = x.new_empty(-(-size // x.element_size()))
    return args[:8 * at] + _TWO.pack(workspace.data_ptr(), size) + args[8 * at + 16:], workspace


def _with_device(device, function, *args):
    """A size query: the answer depends on the device's SM count."""
    if device.index == _current_device():
        return function(*args)
    with _torch_module.cuda.device(device):
        return function(*args)


def _differentiable(*tensors):
    if _torch_module.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                return True
    if _forward_ad._current_level >= 0:                      # (what has no forward derivative says so, in autograd)
        for x in tensors:
            if x is not None and _forward_ad.unpack_dual(x).tangent is not None:
                return True
    return False


def _like(x):
    """A dense tensor of the shape, type and device of x."""
    if x.is_contiguous():
        return _torch_module.empty_like(x)
    return x.new_empty(x.shape)


def _above(grad):
    """A gradient from above as the kernels read it: memory of its own values (it may be a view of negated ones) whose
    innermost axis is contiguous."""
    if grad is None:
        return None
    if grad.is_neg():
        grad = grad.resolve_neg()
    return grad if grad.stride(-1) == 1 else grad.contiguous()


def _dense_above(grad):
    return None if grad is None else _above(grad).contiguous()


def _changed(state):
    """A state that a kernel wrote to: a backward pass that kept it finds out, as with any change in place."""
    if not state.is_inference():
        _torch_module.autograd.graph.increment_version(state)


def _no_gradient(what, *tensors):
    if _differentiable(*tensors):
        raise RuntimeError('%s has no gradient: call it under torch.no_grad()' % what)


def _strides(x, *axes):
    return (0,) * len(axes) if x is None else tuple(x.stride(a) for a in axes)


# ---------------------------------------------------------------------------------------------------------
# selective scan

def _scan_args(dims, x, out=(None, None, None), above=(None, None), grads=(None,) * 9):
    u, delta, A, B, C, D, z, delta_bias, initial_state, lengths = x
    batch, length, channels, states, groups, softplus = dims
    gout, gfinal = above
    gu, gdelta, gA, gB, gC, gD, gz, gbias, ginitial = grads
    return _SCAN.pack(
        _codes[u.dtype], batch, length, channels, states, groups, softplus, u.data_ptr(), delta.data_ptr(), _ptr(z),
        B.data_ptr(), C.data_ptr(), A.data_ptr(), _ptr(D), _ptr(delta_bias), _ptr(initial_state), _ptr(lengths),
        *u.stride()[:2], *delta.stride()[:2], *_strides(z, 0, 1), *B.stride()[:3], *C.stride()[:3],
        _ptr(out[0]), _ptr(out[1]), _ptr(out[2]), 0, 0,
        _ptr(gout), *_strides(gout, 0, 1), _ptr(gfinal), _ptr(gu), _ptr(gdelta), _ptr(gz), _ptr(gB), _ptr(gC), _ptr(gA),
        _ptr(gD), _ptr(gbias), _ptr(ginitial))


def _scan_forward(x, dims, save):
    torch = _torch_module
    u, A = x[0], x[2]
    batch, length, channels, states, _, _ = dims
    device = u.device
    out = _like(u)
    final = A.new_empty((batch, channels, states)) if x[8] is None else torch.empty_like(x[8])
    saved = A.new_empty((batch, (length + 15) // 16, channels, states)) if save else None
    args = _scan_args(dims, x, (out, final, saved))
    size = _with_device(device, launcher.library().ovl_selective_scan_workspace_bytes, args, 0)
    args, workspace = _with_workspace(args, 32, size, u)
    _launch('ovl_selective_scan', args, device)
    return out, final, saved


def _scan_backward(x, dims, saved, gout, gfinal):
    torch = _torch_module
    u, delta, A, B, C, D, z, delta_bias, initial_state, lengths = x
    batch, length, channels, states, groups, _ = dims
    device = u.device
    if gout is None:                                         # only the final state is used further on
        gout = u.new_zeros(channels).expand(batch, length, channels)
    gout, gfinal = _above(gout), _dense_above(gfinal)
    make = torch.zeros_like if batch == 0 else torch.empty_like
    gu, gdelta, gz = _like(u), _like(delta), None if z is None else _like(z)
    gB, gC = _like(B), _like(C)
    gA, gD, gbias = make(A), None if D is None else make(D), None if delta_bias is None else make(delta_bias)
    ginitial = None if initial_state is None else torch.empty_like(initial_state)
    grads = (gu, gdelta, gA, gB, gC, gD, gz, gbias, ginitial)
    args = _scan_args(dims, x, (None, None, saved), (gout, gfinal), grads)
    size = _with_device(device, launcher.library().ovl_selective_scan_workspace_bytes, args, 1)
    args, workspace = _with_workspace(args, 32, size, u)
    _launch('ovl_selective_scan_backward', args, device)
    return grads


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, initial_state=None,
                   lengths=None, return_state=False):
    """The selective scan of a state space layer over whole sequences.

    For every batch, channel ``d`` (of group ``g = d // (channels // groups)``), state ``n`` and token ``t``::

        dt = softplus(delta + delta_bias)                    # delta_softplus=False: delta + delta_bias
        h_t[n] = exp(dt * A[d, n]) * h_{t-1}[n] + dt * u_t * B_t[g, n]
        out_t = (sum_n C_t[g, n] * h_t[n] + D[d] * u_t) * silu(z_t)

    ``u``, ``delta``, ``z``: [batch, length, channels]; ``B``, ``C``: [batch, length, groups, states], or
    [batch, length, states] for one group - all of the type of ``u``.  ``A`` [channels, states], ``D`` and ``delta_bias``
    [channels], ``initial_state`` [batch, channels, states]: float32.  ``D``, ``z``, ``delta_bias`` and ``initial_state``
    may be left out (no skip, no gate, no bias, zeros).  ``lengths`` (int32 [batch], on the device, clamped to
    0 ... length): tokens from ``lengths[b]`` on are padding - never looked at, their outputs and gradients are zeros and
    the state passes them unchanged.  1 to 128 states.

    Returns ``out`` [batch, length, channels] in the type of ``u``; with ``return_state`` also the states after the last
    token of each sequence, float32 [batch, channels, states].  Differentiable with respect to every floating input; for
    the backward pass the states in front of every 16th token are kept (4 * states / 16 bytes per token and channel)."""
    if _front is not None:
        y = _front.selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, lengths)
        if y is not None:
            return y if return_state else y[0]
    what = 'selective_scan'
    torch = _first(u, 'u', 3, what)
    batch, length, channels = u.shape
    t, f32 = u.dtype, torch.float32
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        raise TypeError('%s: A must be a torch tensor with two axes' % what)
    states = A.shape[1]
    if channels < 1 or not 1 <= states <= MAX_STATES:
        raise ValueError('%s: at least one channel and 1 to %d states are supported, not %d and %d'
                         % (what, MAX_STATES, channels, states))
    if isinstance(B, torch.Tensor) and B.dim() == 3:
        B = B.unsqueeze(2)
    if isinstance(C, torch.Tensor) and C.dim() == 3:
        C = C.unsqueeze(2)
    if not isinstance(B, torch.Tensor) or B.dim() != 4:
        raise TypeError('%s: B must be a torch tensor with 3 or 4 axes' % what)
    groups = B.shape[2]
    if groups < 1 or channels % groups:
        raise ValueError('%s: %d channels do not divide into %d groups' % (what, channels, groups))
    u = _tensor(u, 'u', u.shape, t, what)
    delta = _tensor(delta, 'delta', u.shape, t, what)
    z = None if z is None else _tensor(z, 'z', u.shape, t, what)
    B = _tensor(B, 'B', (batch, length, groups, states), t, what)
    C = _tensor(C, 'C', (batch, length, groups, states), t, what)
    A = _dense(A, 'A', (channels, states), f32, what)
    D = None if D is None else _dense(D, 'D', (channels,), f32, what)
    delta_bias = None if delta_bias is None else _dense(delta_bias, 'delta_bias', (channels,), f32, what)
    if initial_state is not None:
        initial_state = _dense(initial_state, 'initial_state', (batch, channels, states), f32, what)
    lengths = _index(lengths, 'lengths', batch, what)
    _one_device(what, u, delta, A, B, C, D, z, delta_bias, initial_state, lengths)
    x = (u, delta, A, B, C, D, z, delta_bias, initial_state, lengths)
    dims = (batch, length, channels, states, groups, 1 if delta_softplus else 0)
    if _differentiable(*x):
        out, final = _autograd().scan.apply(dims, *x)
    else:
        out, final, _ = _scan_forward(x, dims, False)
    return (out, final) if return_state else out


def selective_scan_step(state, u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, slots=None):
    """One token of :func:`selective_scan` for each of many sequences, ``state`` updated in place.

    ``state``: float32 [slots, channels, states], contiguous; ``u``, ``delta``, ``z``: [rows, channels]; ``B``, ``C``:
    [rows, groups, states] or [rows, states].  Row ``r`` keeps its state in slot ``slots[r]`` (int32 [rows], on the
    device), in slot ``r`` without ``slots``.  A negative slot marks a row of padding: its output is zeros.  A slot that
    does not exist, or that an earlier row of the call has already, is left alone and the row's output is NaN.
    Returns [rows, channels] in the type of ``u``.  No gradient."""
    if _front is not None:
        y = _front.selective_scan_step(state, u, delta, A, B, C, D, z, delta_bias, delta_softplus, slots)
        if y is not None:
            return y
    what = 'selective_scan_step'
    torch = _first(u, 'u', 2, what)
    rows, channels = u.shape
    t, f32 = u.dtype, torch.float32
    _state(state, 'state', 3, f32, what)
    n_slots, _, states = state.shape
    if channels < 1 or not 1 <= states <= MAX_STATES:
        raise ValueError('%s: at least one channel and 1 to %d states are supported, not %d and %d'
                         % (what, MAX_STATES, channels, states))
    if state.shape[1] != channels:
        raise ValueError('%s: state has %d channels, u has %d' % (what, state.shape[1], channels))
    if slots is None and n_slots < rows:
        raise ValueError('%s: %d rows but only %d states' % (what, rows, n_slots))
    if isinstance(B, torch.Tensor) and B.dim() == 2:
        B = B.unsqueeze(1)
    if isinstance(C, torch.Tensor) and C.dim() == 2:
        C = C.unsqueeze(1)
    if not isinstance(B, torch.Tensor) or B.dim() != 3:
        raise TypeError('%s: B must be a torch tensor with 2 or 3 axes' % what)
    groups = B.shape[1]
    if groups < 1 or channels % groups:
        raise ValueError('%s: %d channels do not divide into %d groups' % (what, channels, groups))
    u = _tensor(u, 'u', (rows, channels), t, what)
    delta = _tensor(delta, 'delta', (rows, channels), t, what)
    z = None if z is None else _tensor(z, 'z', (rows, channels), t, what)
    B = _tensor(B, 'B', (rows, groups, states), t, what)
    C = _tensor(C, 'C', (rows, groups, states), t, what)
    A = _dense(A, 'A', (channels, states), f32, what)
    D = None if D is None else _dense(D, 'D', (channels,), f32, what)
    delta_bias = None if delta_bias is None else _dense(delta_bias, 'delta_bias', (channels,), f32, what)
    slots = _index(slots, 'slots', rows, what)
    _no_gradient(what, state, u, delta, A, B, C, D, z, delta_bias)
    device = _one_device(what, u, state, delta, A, B, C, D, z, delta_bias, slots)
    out = _like(u)
    _launch('ovl_selective_scan_step', _SCAN_STEP.pack(
        _codes[t], rows, channels, states, groups, 1 if delta_softplus else 0, n_slots, u.data_ptr(), delta.data_ptr(),
        _ptr(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), _ptr(D), _ptr(delta_bias), _ptr(slots), u.stride(0),
        delta.stride(0), 0 if z is None else z.stride(0), B.stride(0), B.stride(1), C.stride(0), C.stride(1),
        state.data_ptr(), out.data_ptr()), device)
    _changed(state)
    return out


# ---------------------------------------------------------------------------------------------------------
# causal convolution

def _activation(activation, what):
    if activation not in (None, 'silu'):
        raise ValueError("%s: activation must be None or 'silu', not %r" % (what, activation))
    return 1 if activation else 0


def _param_type(weight, name, t, what):
    if not isinstance(weight, _torch_module.Tensor):
        raise TypeError('%s: %s must be a torch tensor' % (what, name))
    if weight.dtype is not t and weight.dtype is not _torch_module.float32:
        raise TypeError('%s: %s must be %s or float32, not %s' % (what, name, t, weight.dtype))
    return weight.dtype


def _conv_args(dims, x, out=(None, None), above=(None, None), grads=(None,) * 4):
    x, weight, bias, initial_state, lengths = x
    batch, length, channels, taps, silu = dims
    gout, gfinal = above
    return _CONV.pack(
        _codes[x.dtype], batch, length, channels, taps, silu, weight.dtype is _torch_module.float32, x.data_ptr(),
        weight.data_ptr(), _ptr(bias), _ptr(initial_state), _ptr(lengths), *x.stride()[:2], _ptr(out[0]), _ptr(out[1]),
        _ptr(gout), *_strides(gout, 0, 1), _ptr(gfinal), *map(_ptr, grads), 0, 0)


def _conv_forward(x, dims, state):
    torch = _torch_module
    batch, length, channels, taps, _ = dims
    out = _like(x[0])
    final = None
    if state:
        final = out.new_empty((batch, taps - 1, channels)) if x[3] is None else torch.empty_like(x[3])
    _launch('ovl_causal_conv', _conv_args(dims, x, (out, final)), out.device)
    return out, final


def _conv_backward(x, dims, gout, gfinal):
    torch = _torch_module
    batch, length, channels, taps, _ = dims
    tokens, weight, bias, initial_state, _ = x
    device = tokens.device
    if gout is None:
        gout = tokens.new_zeros(channels).expand(batch, length, channels)
    gout, gfinal = _above(gout), _dense_above(gfinal)
    make = torch.zeros_like if batch == 0 else torch.empty_like
    gx, gweight, gbias = _like(tokens), make(weight), None if bias is None else make(bias)
    ginitial = None if initial_state is None else torch.empty_like(initial_state)
    grads = (gx, gweight, gbias, ginitial)
    args = _conv_args(dims, x, (None, None), (gout, gfinal), grads)
    size = _with_device(device, launcher.library().ovl_causal_conv_workspace_bytes, args)
    args, workspace = _with_workspace(args, 24, size, tokens)
    _launch('ovl_causal_conv_backward', args, device)
    return grads


def causal_conv1d(x, weight, bias=None, activation=None, initial_state=None, lengths=None, return_state=False):
    """Causal convolution along the tokens, every channel by itself::

        out_t[d] = act(bias[d] + sum_k weight[d, k] * x_{t - (taps - 1) + k}[d])

    ``x``: [batch, length, channels]; ``weight``: [channels, taps], ``bias``: [channels], both in the type of ``x`` or
    both float32; 1 to 8 taps; ``activation``: None or 'silu'.  ``initial_state`` [batch, taps - 1, channels], in the type
    of ``x``: the inputs in front of the first token (zeros without it).  ``lengths`` as for :func:`selective_scan`.

    Returns [batch, length, channels]; with ``return_state`` also the last ``taps - 1`` inputs of each sequence (those of
    ``initial_state`` among them when it is shorter), [batch, taps - 1, channels].  Differentiable with respect to ``x``,
    ``weight``, ``bias`` and ``initial_state``."""
    if _front is not None:
        y = _front.causal_conv1d(x, weight, bias, activation, initial_state, lengths, return_state)
        if y is not None:
            return y if return_state else y[0]
    what = 'causal_conv1d'
    torch = _first(x, 'x', 3, what)
    batch, length, channels = x.shape
    t = x.dtype
    silu = _activation(activation, what)
    p = _param_type(weight, 'weight', t, what)
    if weight.dim() != 2 or channels < 1 or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError('%s: weight must be [channels, taps] with at least one channel and 1 to %d taps'
                         % (what, MAX_TAPS))
    taps = weight.shape[1]
    x = _tensor(x, 'x', x.shape, t, what)
    weight = _dense(weight, 'weight', (channels, taps), p, what)
    bias = None if bias is None else _dense(bias, 'bias', (channels,), p, what)
    if initial_state is not None:
        initial_state = _dense(initial_state, 'initial_state', (batch, taps - 1, channels), t, what)
    lengths = _index(lengths, 'lengths', batch, what)
    _one_device(what, x, weight, bias, initial_state, lengths)
    args, dims = (x, weight, bias, initial_state, lengths), (batch, length, channels, taps, silu)
    if _differentiable(*args):
        out, final = _autograd().conv.apply(dims, return_state, *args)
    else:
        out, final = _conv_forward(args, dims, return_state)
    return (out, final) if return_state else out


def causal_conv1d_step(state, x, weight, bias=None, activation=None, slots=None):
    """One token of :func:`causal_conv1d` for each of many sequences, ``state`` shifted in place.

    ``state``: [slots, taps - 1, channels] in the type of ``x``, contiguous: the last ``taps - 1`` inputs of each sequence;
    ``x``: [rows, channels].  ``slots`` as for :func:`selective_scan_step`.  Returns [rows, channels].  No gradient."""
    if _front is not None:
        y = _front.causal_conv1d_step(state, x, weight, bias, activation, slots)
        if y is not None:
            return y
    what = 'causal_conv1d_step'
    torch = _first(x, 'x', 2, what)
    rows, channels = x.shape
    t = x.dtype
    silu = _activation(activation, what)
    _state(state, 'state', 3, t, what)
    p = _param_type(weight, 'weight', t, what)
    if weight.dim() != 2 or channels < 1 or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError('%s: weight must be [channels, taps] with at least one channel and 1 to %d taps'
                         % (what, MAX_TAPS))
    taps = weight.shape[1]
    if state.shape[1] != taps - 1 or state.shape[2] != channels:
        raise ValueError('%s: state must have the shape (slots, %d, %d), not %s'
                         % (what, taps - 1, channels, tuple(state.shape)))
    if slots is None and state.shape[0] < rows:
        raise ValueError('%s: %d rows but only %d states' % (what, rows, state.shape[0]))
    x = _tensor(x, 'x', (rows, channels), t, what)
    weight = _dense(weight, 'weight', (channels, taps), p, what)
    bias = None if bias is None else _dense(bias, 'bias', (channels,), p, what)
    slots = _index(slots, 'slots', rows, what)
    _no_gradient(what, state, x, weight, bias)
    device = _one_device(what, x, state, weight, bias, slots)
    out = _like(x)
    _launch('ovl_causal_conv_step', _CONV_STEP.pack(
        _codes[t], rows, channels, taps, silu, p is torch.float32, state.shape[0], x.data_ptr(), weight.data_ptr(),
        _ptr(bias), _ptr(slots), x.stride(0), state.data_ptr(), out.data_ptr()), device)
    _changed(state)
    return out


# ---------------------------------------------------------------------------------------------------------
# root-mean-square norm

def _rows(x):
    """[..., columns] as [rows, columns] (a view where the strides allow it)."""
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def _norm_args(x, weight, eps, group=0, residual=None, y=None, residual_out=None, q=None, scale=None, gy=None, gres=None,
               gx=None, gweight=None):
    return _NORM.pack(
        _codes[x.dtype], x.shape[0], x.shape[1], weight.dtype is _torch_module.float32, group, eps, x.data_ptr(),
        _ptr(residual), weight.data_ptr(), x.stride(0), 0 if residual is None else residual.stride(0), _ptr(y),
        _ptr(residual_out), _ptr(q), _ptr(scale), _ptr(gy), _ptr(gres), 0 if gy is None else gy.stride(0),
        0 if gres is None else gres.stride(0), _ptr(gx), _ptr(gweight), 0, 0)


def _norm_check(x, weight, residual, eps, what):
    _first(x, 'x', None, what)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_COLUMNS:
        raise ValueError('%s: x must have 1 to %d columns' % (what, MAX_COLUMNS))
    if not isinstance(eps, (int, float)) or isinstance(eps, bool) or not 0 <= eps < float('inf'):
        raise ValueError('%s: eps must be a number that is not negative' % what)
    weight = _dense(weight, 'weight', (x.shape[-1],), _param_type(weight, 'weight', x.dtype, what), what)
    if residual is not None:
        residual = _tensor(residual, 'residual', x.shape, x.dtype, what)
    x = _tensor(x, 'x', x.shape, x.dtype, what)
    device = _one_device(what, x, weight, residual)
    return x, weight, residual, float(eps), device


def _norm_forward(x, weight, residual, eps):
    x, residual = _rows(x), None if residual is None else _rows(residual)
    y = _like(x)
    residual_out = None if residual is None else _like(x)
    _launch('ovl_rms_norm', _norm_args(x, weight, eps, 0, residual, y, residual_out), x.device)
    return y, residual_out


def _norm_backward(x, weight, residual, eps, gy, gres):
    torch = _torch_module
    device = x.device
    if gy is None:
        gy = x.new_zeros(x.shape[1]).expand(x.shape)
    gy, gres = _above(gy), _above(gres)
    gx = _like(x)
    gweight = torch.empty_like(weight)
    args = _norm_args(x, weight, eps, residual=residual, gy=gy, gres=gres, gx=gx, gweight=gweight)
    size = _with_device(device, launcher.library().ovl_rms_norm_workspace_bytes, args)
    args, workspace = _with_workspace(args, 21, size, x)
    _launch('ovl_rms_norm_backward', args, device)
    return gx, gweight


def rms_norm(x, weight, residual=None, eps=1e-6):
    """Root-mean-square norm over the last axis, with the residual's addition in front of it::

        s = x + residual;  y = s / sqrt(mean(s^2) + eps) * weight

    ``x``, ``residual``: [..., columns] of one type, 1 to 32768 columns; ``weight``: [columns], in that type or float32.
    Returns ``y``, with a ``residual`` the pair ``(y, s)``: ``s`` rounded to the type of ``x`` is the residual of the next
    block (the norm itself, and its gradient, use the unrounded sum).  Differentiable with respect to all three."""
    if _front is not None:
        y = _front.rms_norm(x, weight, residual, eps)
        if y is not None:
            return y[0] if residual is None else y
    x, weight, residual, eps, _ = _norm_check(x, weight, residual, eps, 'rms_norm')
    if _differentiable(x, weight, residual):
        y, residual_out = _autograd().norm.apply(x, weight, residual, eps)
    else:
        y, residual_out = _norm_forward(x, weight, residual, eps)
        if x.dim() != 2:
            y = y.view(x.shape)
            residual_out = None if residual_out is None else residual_out.view(x.shape)
    return y if residual is None else (y, residual_out)


def rms_norm_quantize(x, weight, residual=None, eps=1e-6, group=None):
    """:func:`rms_norm` with an output in 8 bits.  The row is cut into groups of ``group`` columns (which divides the
    number of columns; None: the whole row), each with a scale::

        scale = max(max |y| / 448, 2^-126);  q = y / scale, rounded to the nearest e4m3 value

    Returns ``(q, scale)``, with a ``residual`` ``(q, scale, s)``: ``q`` float8_e4m3fn in the shape of ``x``, ``scale``
    float32 [..., columns / group].  Both quotients are rounded to 32 bits as a division does.  A group whose ``y`` has a NaN
    is NaN as a whole (an infinity of ``x`` or ``residual`` makes one); an infinite weight makes its group's scale infinite,
    the infinite value NaN and the others zeros.  No gradient."""
    if _front is not None:
        y = _front.rms_norm(x, weight, residual, eps, group)
        if y is not None:
            return y
    what = 'rms_norm_quantize'
    x, weight, residual, eps, device = _norm_check(x, weight, residual, eps, what)
    torch, columns = _torch_module, x.shape[-1]
    group = columns if group is None else group
    if not isinstance(group, int) or isinstance(group, bool) or group < 1 or columns % group:
        raise ValueError('%s: group must divide the %d columns, not %r' % (what, columns, group))
    _no_gradient(what, x, weight, residual)
    shape, x, residual = x.shape, _rows(x), None if residual is None else _rows(residual)
    q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    scale = x.new_empty((x.shape[0], columns // group), dtype=torch.float32)
    residual_out = None if residual is None else _like(x)
    _launch('ovl_rms_norm', _norm_args(x, weight, eps, group, residual, None, residual_out, q, scale), device)
    if len(shape) != 2:
        q, scale = q.view(shape), scale.view(shape[:-1] + (columns // group,))
        residual_out = None if residual is None else residual_out.view(shape)
    return (q, scale) if residual is None else (q, scale, residual_out)


# ---------------------------------------------------------------------------------------------------------
# autograd

_functions = None


def _autograd():
    """The autograd functions, made on first use (torch is imported lazily by this package)."""
    global _functions
    if _functions is not None:
        return _functions
    import types
    torch = _torch()

    def once_differentiable(backward):
        """Gradients that are differentiated again (create_graph) say so instead of counting as constants, whether or not
        the gradient above is one of them."""
        def call(ctx, *above):
            with torch.no_grad():
                grads = backward(ctx, *above)
            if not torch.is_grad_enabled():
                return grads
            error = torch._C._functions.DelayedError('the sequence operators are differentiable once', len(grads))
            return error(*(None if g is None else g.detach().requires_grad_() for g in grads))
        return call

    class SelectiveScan(torch.autograd.Function):
        @staticmethod
        def forward(ctx, dims, *x):
            out, final, saved = _scan_forward(x, dims, True)
            ctx.dims = dims
            ctx.save_for_backward(*x, saved)
            ctx.set_materialize_grads(False)
            return out, final

        @staticmethod
        @once_differentiable
        def backward(ctx, gout, gfinal):
            if gout is None and gfinal is None:
                return (None,) * 11
            *x, saved = ctx.saved_tensors
            gu, gdelta, gA, gB, gC, gD, gz, gbias, ginitial = _scan_backward(x, ctx.dims, saved, gout, gfinal)
            return None, gu, gdelta, gA, gB, gC, gD, gz, gbias, ginitial, None

    class CausalConv(torch.autograd.Function):
        @staticmethod
        def forward(ctx, dims, state, *x):
            out, final = _conv_forward(x, dims, state)
            ctx.dims = dims
            ctx.save_for_backward(*x)
            ctx.set_materialize_grads(False)
            return out, final

        @staticmethod
        @once_differentiable
        def backward(ctx, gout, gfinal):
            if gout is None and gfinal is None:
                return (None,) * 7
            return (None, None) + _conv_backward(ctx.saved_tensors, ctx.dims, gout, gfinal) + (None,)

    class RmsNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, residual, eps):
            y, residual_out = _norm_forward(x, weight, residual, eps)
            y = y.view(x.shape)
            residual_out = None if residual_out is None else residual_out.view(x.shape)
            ctx.eps = eps
            ctx.save_for_backward(x, weight, residual)
            ctx.set_materialize_grads(False)
            return y, residual_out

        @staticmethod
        @once_differentiable
        def backward(ctx, gy, gres):
            if gy is None and gres is None:
                return None, None, None, None
            x, weight, residual = ctx.saved_tensors
            gx, gweight = _norm_backward(_rows(x), weight, None if residual is None else _rows(residual), ctx.eps,
                                         None if gy is None else _rows(gy), None if gres is None else _rows(gres))
            gx = gx.view(x.shape)
            return gx, gweight, gx if ctx.needs_input_grad[2] else None, None

    _functions = types.SimpleNamespace(scan=SelectiveScan, conv=CausalConv, norm=RmsNorm)
    return _functions
