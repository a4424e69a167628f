"""Plain float64 statements of the sequence operators (selective scan, short causal convolution, root-mean-square norm),
token after token as they are defined, on any device.  Gradients come from autograd over these statements."""
import torch


def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def silu(x):
    return x / (1 + torch.exp(-x))


def per_channel(x, channels):
    """[batch, groups, states] -> [batch, channels, states]"""
    return x.repeat_interleave(channels // x.shape[1], 1)


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, initial_state=None, lengths=None,
         magnitude=False):
    """(outputs, final state); padding: outputs 0, state unchanged.  ``magnitude``: with the absolute values of all other
    factors as arguments, the sums of the terms' magnitudes (a step size counts as it is in the decay only)."""
    batch, length, channels = u.shape
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    h = u.new_zeros(batch, channels, A.shape[1]) if initial_state is None else initial_state
    ends = torch.full((batch,), length, device=u.device) if lengths is None else lengths.long().clamp(0, length)
    outs = []
    for t in range(length):
        on = (t < ends)[:, None]
        dt = delta[:, t] if delta_bias is None else delta[:, t] + delta_bias
        dt = softplus(dt) if delta_softplus else dt
        ut, Bt, Ct = u[:, t], per_channel(B[:, t], channels), per_channel(C[:, t], channels)
        # padding may hold anything, infinities and NaN too: it is put aside before it meets the state
        dt, ut = torch.where(on, dt, 0.0), torch.where(on, ut, 0.0)
        Bt, Ct = torch.where(on[..., None], Bt, 0.0), torch.where(on[..., None], Ct, 0.0)
        h = torch.exp(dt[..., None] * A) * h + ((dt.abs() if magnitude else dt) * ut)[..., None] * Bt
        y = (h * Ct).sum(-1)
        if D is not None:
            y = y + D * ut
        if z is not None:
            y = y * silu(torch.where(on, z[:, t], 0.0))
        outs.append(torch.where(on, y, 0.0))
    return (torch.stack(outs, 1) if outs else u.clone()), h


def conv(x, weight, bias=None, activation=None, initial_state=None, lengths=None):
    batch, length, channels = x.shape
    taps = weight.shape[1]
    state = x.new_zeros(batch, taps - 1, channels) if initial_state is None else initial_state
    outs, finals = [], []
    for b in range(batch):
        end = length if lengths is None else max(0, min(int(lengths[b]), length))
        xs = torch.cat([state[b], x[b, :end]])
        y = sum(weight[:, k] * xs[k:k + end] for k in range(taps))
        if bias is not None:
            y = y + bias
        y = silu(y) if activation == 'silu' else y
        outs.append(torch.cat([y, x.new_zeros(length - end, channels)]))
        finals.append(xs[end:])
    return torch.stack(outs), torch.stack(finals)


def rms_norm(x, weight, residual=None, eps=1e-6):
    s = x if residual is None else x + residual
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * weight
    return y, s


def e4m3(v):
    """The nearest value with three bits behind the leading one and exponents from -6 on, ties to even."""
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))), min=-6) - 3)
    return torch.round(v / unit) * unit


def rms_norm_quantize(x, weight, residual=None, eps=1e-6, group=None):
    """(scaled values before rounding, scales, sum)"""
    y, s = rms_norm(x, weight, residual, eps)
    parts = y.unflatten(-1, (-1, group or x.shape[-1]))
    scale = torch.clamp(parts.abs().amax(-1) / 448, min=2.0 ** -126)
    return (parts / scale[..., None]).flatten(-2), scale, s
