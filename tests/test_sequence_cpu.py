"""The sequence operators without a device: what they refuse, and that they say so before anything is launched."""
import os
import re

import pytest
import torch

import opveclib_b200 as ovl
import sequence_reference as ref
from opveclib_b200 import launcher, sequence

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32 = torch.bfloat16, torch.float32


def _scan_inputs(batch=2, length=5, channels=6, states=4, groups=2, t=BF16):
    return dict(u=torch.zeros(batch, length, channels, dtype=t), delta=torch.zeros(batch, length, channels, dtype=t),
                A=torch.zeros(channels, states), B=torch.zeros(batch, length, groups, states, dtype=t),
                C=torch.zeros(batch, length, groups, states, dtype=t))


def _step_inputs(rows=2, channels=6, states=4, groups=2, t=BF16):
    return dict(state=torch.zeros(rows, channels, states), u=torch.zeros(rows, channels, dtype=t),
                delta=torch.zeros(rows, channels, dtype=t), A=torch.zeros(channels, states),
                B=torch.zeros(rows, groups, states, dtype=t), C=torch.zeros(rows, groups, states, dtype=t))


@pytest.mark.parametrize('change, error', [
    (dict(u=[1.0]), TypeError), (dict(u=torch.zeros(2, 5, 6, dtype=torch.float64)), TypeError),
    (dict(u=torch.zeros(5, 6, dtype=BF16)), ValueError), (dict(delta=torch.zeros(2, 5, 6)), TypeError),
    (dict(delta=torch.zeros(2, 5, 7, dtype=BF16)), ValueError), (dict(A=torch.zeros(6, 4, dtype=BF16)), TypeError),
    (dict(A=torch.zeros(5, 4)), ValueError), (dict(A=torch.zeros(6, 129)), ValueError), (dict(A=torch.zeros(6, 0)), ValueError),
    (dict(B=torch.zeros(2, 5, 2, 3, dtype=BF16)), ValueError), (dict(B=torch.zeros(2, 5, 4, 4, dtype=BF16)), ValueError),
    (dict(B=torch.zeros(2, 5, 2, 4)), TypeError), (dict(C=torch.zeros(2, 5, 1, 4, dtype=BF16)), ValueError),
    (dict(B=None), TypeError), (dict(D=torch.zeros(6, dtype=BF16)), TypeError), (dict(D=torch.zeros(5)), ValueError),
    (dict(z=torch.zeros(2, 4, 6, dtype=BF16)), ValueError), (dict(z=torch.zeros(2, 5, 6)), TypeError),
    (dict(delta_bias=torch.zeros(6, dtype=BF16)), TypeError), (dict(initial_state=torch.zeros(2, 6, 4, dtype=BF16)), TypeError),
    (dict(initial_state=torch.zeros(2, 6, 5)), ValueError), (dict(lengths=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(lengths=[5, 5]), TypeError),
    (dict(), RuntimeError),                                    # everything is right but the device
])
def test_selective_scan_refuses(change, error):
    with pytest.raises(error):
        ovl.selective_scan(**{**_scan_inputs(), **change})


@pytest.mark.parametrize('change, error', [
    (dict(state=torch.zeros(2, 6, 4, dtype=BF16)), TypeError), (dict(state=torch.zeros(1, 6, 4)), ValueError),
    (dict(state=torch.zeros(2, 5, 4)), ValueError), (dict(state=torch.zeros(2, 4, 6).transpose(1, 2)), ValueError),
    (dict(state=torch.zeros(6, 4)), ValueError), (dict(state=None), TypeError), (dict(u=torch.zeros(2, 1, 6, dtype=BF16)), ValueError),
    (dict(B=torch.zeros(2, 4, 4, dtype=BF16)), ValueError), (dict(slots=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(slots=torch.zeros(1, dtype=torch.int32)), ValueError), (dict(D=torch.zeros(6).requires_grad_()), RuntimeError),
    (dict(), RuntimeError),
])
def test_selective_scan_step_refuses(change, error):
    with pytest.raises(error):
        ovl.selective_scan_step(**{**_step_inputs(), **change})


@pytest.mark.parametrize('change, error', [
    (dict(x=torch.zeros(5, 6, dtype=BF16)), ValueError), (dict(x=torch.zeros(2, 5, 6, dtype=torch.int32)), TypeError),
    (dict(weight=torch.zeros(6, 9, dtype=BF16)), ValueError), (dict(weight=torch.zeros(6, 0, dtype=BF16)), ValueError),
    (dict(weight=torch.zeros(5, 4, dtype=BF16)), ValueError), (dict(weight=torch.zeros(6, 4, dtype=torch.float16)), TypeError),
    (dict(bias=torch.zeros(6)), TypeError), (dict(bias=torch.zeros(5, dtype=BF16)), ValueError),
    (dict(activation='relu'), ValueError), (dict(activation=True), ValueError),
    (dict(initial_state=torch.zeros(2, 4, 6, dtype=BF16)), ValueError), (dict(initial_state=torch.zeros(2, 3, 6)), TypeError),
    (dict(lengths=torch.zeros(2)), TypeError), (dict(), RuntimeError),
])
def test_causal_conv1d_refuses(change, error):
    with pytest.raises(error):
        ovl.causal_conv1d(**{**dict(x=torch.zeros(2, 5, 6, dtype=BF16), weight=torch.zeros(6, 4, dtype=BF16)), **change})


@pytest.mark.parametrize('change, error', [
    (dict(state=torch.zeros(2, 3, 6)), TypeError), (dict(state=torch.zeros(2, 4, 6, dtype=BF16)), ValueError),
    (dict(state=torch.zeros(2, 6, 3, dtype=BF16).transpose(1, 2)), ValueError), (dict(state=torch.zeros(1, 3, 6, dtype=BF16)), ValueError),
    (dict(x=torch.zeros(2, 7, dtype=BF16)), ValueError), (dict(weight=torch.zeros(6, 4, dtype=BF16).requires_grad_()), RuntimeError),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(), RuntimeError),
])
def test_causal_conv1d_step_refuses(change, error):
    with pytest.raises(error):
        ovl.causal_conv1d_step(**{**dict(state=torch.zeros(2, 3, 6, dtype=BF16), x=torch.zeros(2, 6, dtype=BF16),
                                         weight=torch.zeros(6, 4, dtype=BF16)), **change})


@pytest.mark.parametrize('change, error', [
    (dict(x=torch.zeros(3, 0)), ValueError), (dict(x=torch.zeros(3, 32769)), ValueError), (dict(x=torch.zeros(())), ValueError),
    (dict(x=torch.zeros(3, 8, dtype=torch.int8)), TypeError), (dict(weight=torch.zeros(7)), ValueError),
    (dict(weight=torch.zeros(8, dtype=BF16)), TypeError), (dict(residual=torch.zeros(3, 7)), ValueError),
    (dict(residual=torch.zeros(3, 8, dtype=BF16)), TypeError), (dict(eps=-1.0), ValueError), (dict(eps=float('nan')), ValueError),
    (dict(eps='1'), ValueError), (dict(eps=True), ValueError), (dict(), RuntimeError),
])
def test_rms_norm_refuses(change, error):
    args = {**dict(x=torch.zeros(3, 8), weight=torch.zeros(8)), **change}
    with pytest.raises(error):
        ovl.rms_norm(**args)
    with pytest.raises(error):
        ovl.rms_norm_quantize(**args)


def test_argument_structures_match_their_packers():
    text = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'ovl_b200.h')).read(), flags=re.S)
    for name, packer in (('OvlSelectiveScan', sequence._SCAN), ('OvlSelectiveScanStep', sequence._SCAN_STEP),
                         ('OvlCausalConv', sequence._CONV), ('OvlCausalConvStep', sequence._CONV_STEP),
                         ('OvlRmsNorm', sequence._NORM)):
        body = re.search(r'typedef struct %s \{(.*?)\} %s;' % (name, name), text, re.S).group(1)
        fields = sum(len(line.split(',')) for line in body.split(';') if line.strip())
        assert packer.size == 8 * fields, name


def _scan_bytes(**change):
    values = dict(dtype=12, batch=1, length=4, channels=8, states=4, groups=1)
    values.update(change)
    head = [values[k] for k in ('dtype', 'batch', 'length', 'channels', 'states', 'groups')]
    return sequence._SCAN.pack(*head, *([0] * (sequence._SCAN.size // 8 - 6)))


@pytest.mark.parametrize('change, status', [
    (dict(dtype=3), 3), (dict(dtype=0), 3), (dict(channels=0), 11), (dict(channels=7, groups=2), 11), (dict(states=129), 10),
    (dict(states=0), 11), (dict(length=-1), 11), (dict(batch=-1), 11), (dict(), 4), (dict(batch=0), 0),
])
def test_entry_points_check_before_any_launch(change, status):
    lib = launcher.library()
    args = _scan_bytes(**change)
    assert lib.ovl_selective_scan(args, None) == status
    assert lib.ovl_selective_scan_backward(args, None) == status
    if status not in (0, 4):
        assert lib.ovl_selective_scan_workspace_bytes(args, 1) == 0


def test_entry_points_refuse_null_and_missing_workspaces():
    lib = launcher.library()
    for name in ('ovl_selective_scan', 'ovl_selective_scan_backward', 'ovl_selective_scan_step', 'ovl_causal_conv',
                 'ovl_causal_conv_backward', 'ovl_causal_conv_step', 'ovl_rms_norm', 'ovl_rms_norm_backward'):
        assert getattr(lib, name)(None, None) == 4, name
    # conv: 12 leading fields, then strides; a backward call without its workspace
    p = 4096
    conv = sequence._CONV.pack(2, 1, 4, 8, 4, 0, 0, p, p, 0, 0, 0, 32, 8, 0, 0, p, 32, 8, 0, p, p, 0, 0, 0, 0)
    assert lib.ovl_causal_conv_workspace_bytes(conv) > 0
    assert lib.ovl_causal_conv_backward(conv, None) == 7
    norm = sequence._NORM.pack(2, 4, 8, 0, 0, 1e-6, p, 0, p, 8, 0, 0, 0, 0, 0, p, 0, 8, 0, p, p, 0, 0)
    assert lib.ovl_rms_norm_workspace_bytes(norm) > 0
    assert lib.ovl_rms_norm_backward(norm, None) == 7
    # a group that does not divide the columns, more columns than a row may have
    assert lib.ovl_rms_norm(sequence._NORM.pack(2, 4, 8, 0, 3, 1e-6, *([0] * 17)), None) == 11
    assert lib.ovl_rms_norm(sequence._NORM.pack(2, 4, 32769, 0, 0, 1e-6, *([0] * 17)), None) == 10
    # fewer states than rows
    step = [12, 4, 8, 4, 1, 0, 3] + [p] * 8 + [0] * 10
    assert lib.ovl_selective_scan_step(sequence._SCAN_STEP.pack(*(step[:14] + [0] + step[15:])), None) == 11


def test_work_space_grows_with_the_problem_and_is_none_for_many_channels():
    lib = launcher.library()
    assert lib.ovl_selective_scan_workspace_bytes(_scan_bytes(batch=64, length=64, channels=4096, states=16), 0) == 0
    few = lib.ovl_selective_scan_workspace_bytes(_scan_bytes(length=4096, channels=64, states=16), 0)
    assert few > 0                                             # the length is cut into segments
    assert lib.ovl_selective_scan_workspace_bytes(_scan_bytes(length=4096, channels=64, states=16), 1) > few


def test_the_reference_statements_themselves():
    """The float64 statements that the device tests compare with, against hand-computed values."""
    out, h = ref.scan(torch.tensor([[[2.0], [3.0]]]).double(), torch.tensor([[[1.0], [0.5]]]).double(),
                      torch.tensor([[0.0]]).double(), torch.ones(1, 2, 1).double(), torch.ones(1, 2, 1).double())
    assert out.flatten().tolist() == [2.0, 3.5] and h.item() == 3.5
    out, state = ref.conv(torch.arange(1.0, 4.0).view(1, 3, 1), torch.tensor([[10.0, 1.0]]))
    assert out.flatten().tolist() == [1.0, 12.0, 23.0] and state.item() == 3.0
    assert ref.e4m3(torch.tensor([17.0, 18.0, 19.0, 0.001, 449.0]).double()).tolist()[:3] == [16.0, 18.0, 20.0]


# ---- the compiled way of the usual calls --------------------------------------------------------------

def test_the_compiled_way_hands_back_what_is_not_its_own():
    """Without a device every call is one that sequence.py has to refuse; nothing is launched, nothing raised."""
    import importlib.util
    from opveclib_b200 import compiler
    path = compiler.build_front()
    if path is None:
        pytest.skip('no C++ compiler')
    spec = importlib.util.spec_from_file_location('ovl_front', path)
    front = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(front)
    x, w = torch.randn(4, 16), torch.ones(16)
    for call, args in ((front.rms_norm, (x, w, None, 1e-6)), (front.rms_norm, ()), (front.rms_norm, (x, w, None, 1e-6, 8, 8)),
                       (front.rms_norm, (torch.nn.Parameter(x), w, None, 1e-6, None)), (front.selective_scan, (1, 2)),
                       (front.selective_scan, (None,) * 11), (front.selective_scan_step, (x,) * 11),
                       (front.causal_conv1d, (x,) * 7), (front.causal_conv1d_step, (x,) * 6), (front.causal_conv1d_step, ())):
        assert call(*args) is None
    for bad in ((), (torch.nn.Parameter,), (torch.nn.Parameter,) + (0,) * 11, (torch.nn.Parameter,) + ('x',) * 11):
        with pytest.raises((TypeError, ValueError)):
            front.bind(*bad)


def test_a_module_that_cannot_be_built_is_done_without(monkeypatch, caplog):
    from opveclib_b200 import compiler, sequence

    def fails(force=False):
        raise RuntimeError('no headers')
    monkeypatch.setattr(compiler, 'build_front', fails)
    monkeypatch.setattr(sequence, '_front', None)
    monkeypatch.setattr(sequence, '_front_tried', False)
    sequence._load_front()
    assert sequence._front is None and sequence._front_tried


@pytest.mark.parametrize('tracer', ['jit', 'fx', 'fx before dispatch', 'export'])
def test_tracing_is_refused_before_the_arguments_are_looked_at(tracer):
    """A tracer would keep the example's answer (tests/test_sequence_calls_gpu.py has the calls on a device)."""
    from torch.fx.experimental.proxy_tensor import make_fx
    w, taps, state = torch.ones(8), torch.ones(8, 4), torch.zeros(2, 8, 4)
    A, B = -torch.ones(8, 4), torch.ones(2, 5, 4)

    def by(call, x):
        if tracer == 'jit':
            torch.jit.trace(call, (x,), check_trace=False)
        elif tracer == 'export':
            module = torch.nn.Module()
            module.forward = call
            torch.export.export(module, (x,), strict=False)
        else:
            make_fx(call, pre_dispatch=tracer != 'fx')(x)
    x = torch.zeros(2, 5, 8)
    for call, arg in ((lambda v: ovl.rms_norm(v * 2, w), x), (lambda v: ovl.rms_norm_quantize(v * 2, w)[1], x),
                      (lambda v: ovl.causal_conv1d(v * 2, taps), x), (lambda v: ovl.selective_scan(v, v * 2, A, B, B), x),
                      (lambda v: ovl.causal_conv1d_step(torch.zeros(2, 3, 8), v * 2, taps), x[:, 0]),
                      (lambda v: ovl.selective_scan_step(state, v, v * 2, A, B[:, 0], B[:, 0]), x[:, 0])):
        with pytest.raises(RuntimeError, match='cannot be traced'):
            by(call, arg)
    with pytest.raises(RuntimeError, match='needs CUDA tensors'):           # and is over with the tracer
        ovl.rms_norm(x, w)


@pytest.mark.parametrize('batch, length, channels, states, groups', [(8, 4096, 4096, 128, 1), (4, 2048, 4096, 128, 1), (1, 16384, 8192, 64, 1),
                                                                     (2, 4096, 8192, 100, 2), (64, 2048, 2048, 65, 1), (1, 8192, 16384, 33, 4)])
def test_the_work_space_of_many_states_is_bounded(batch, length, channels, states, groups):
    """The parts of gB and gC once took 8 bytes per token, padded state and tile of 4 to 8 channels: 34 GB for the first
    case.  Now 1 GB, or what the blocks that run at a time leave (at most 2 on each of 148 SMs, and up to twice that by
    rounding up), beside their sum and the parameters' parts."""
    lib = launcher.library()
    args = _scan_bytes(batch=batch, length=length, channels=channels, states=states, groups=groups)
    padded = 64 if states <= 64 else 128
    at_a_time = (148 + batch * groups) * (2 if states <= 64 else 1) * length * 2 * padded * 4
    others = batch * groups * length * 2 * padded * 4 + 8 * batch * channels * (states + 2) * 4
    assert 0 < lib.ovl_selective_scan_workspace_bytes(args, 1) <= max(1 << 30, at_a_time) + others
