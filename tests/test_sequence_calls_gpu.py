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
