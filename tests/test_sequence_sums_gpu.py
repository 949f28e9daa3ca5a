"""GPU: long sums of the sequence operators' parameter gradients.

Terms 1, e, e, e, ... with e = 2^-25: a sum in float32 that began with the 1 loses every e (1 + e rounds to 1), in any
order of the others.  All products are exact (factors 1), so a gradient is off by the roundings of its own sum alone: at most 512 in
a chain of float32 adds, one where the chain's end is stored, a few inside a workgroup and one of the result, 530 u of the magnitudes,
u = 2^-24, however many rows there are."""

import pytest
import torch

from isaaclab_amd.utils import sequence as S

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -24, 2.0 ** -25


def ones(dev, dtype, *shape):
    return torch.ones((1,) * len(shape), dtype=dtype, device=dev).expand(shape)


def check(got, want, what, units=530):
    off = (got.double().cpu() - want).abs().max()
    assert off <= units * U * want, f"{what}: off by {float(off / want / U):.0f} u"


def test_convolution_of_many_rows(dev):
    """2^31 rows of one channel: 8192 to a thread if 1024 workgroups shared them."""
    batch, length = 256, 2 ** 23
    x = ones(dev, torch.bfloat16, batch, length, 1)
    weight, bias = torch.ones(1, 1, device=dev, requires_grad=True), torch.zeros(1, device=dev, requires_grad=True)
    grad = torch.full((batch, length, 1), E, dtype=torch.bfloat16, device=dev)
    grad[:2, ::64] = 1.0
    want = 2 * length / 64 + (batch * length - 2 * length / 64) * E
    out = S.short_convolution(x, weight, bias)
    for name, g in zip(("weight", "bias"), torch.autograd.grad(out, (weight, bias), grad)):
        check(g, want, name)
