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


def test_recurrence_of_many_sequences(dev):
    """4096 sequences of one row to a workgroup: dA, dD and d delta_bias are each the sum of the output's gradients."""
    batch, channels = 4096, 64 * 1536
    x = ones(dev, torch.bfloat16, batch, 1, channels)
    bc = ones(dev, torch.bfloat16, batch, 1, 1, 1)
    leaves = dict(A=torch.zeros(channels, 1, device=dev), D=torch.ones(channels, device=dev), delta_bias=torch.zeros(channels, device=dev))
    leaves = {k: t.requires_grad_(True) for k, t in leaves.items()}
    grad = torch.full((batch, 1, channels), E, dtype=torch.bfloat16, device=dev)
    grad[0] = 1.0
    out = S.state_space_scan(x, x, leaves["A"], bc, bc, D=leaves["D"], delta_bias=leaves["delta_bias"], softplus=False,
                             state=torch.ones(batch, 1, channels, device=dev))
    for name, g in zip(leaves, torch.autograd.grad(out, tuple(leaves.values()), grad)):
        check(g, 1 + (batch - 1) * E, name)


@pytest.mark.parametrize("with_lengths", [False, True])
def test_recurrence_of_many_rows(dev, with_lengths):
    """Sequences of 16384 and fewer rows, undivided, and workgroups whose sequences end early: dD (a lane adds every fourth row)."""
    batch, length, channels = 12, 2 ** 14, 64 * 160   # two sequences to a workgroup, 64 rows of partial sums
    x = ones(dev, torch.bfloat16, batch, length, channels)
    bc, zero = ones(dev, torch.bfloat16, batch, length, 1, 1), torch.zeros(1, 1, 1, dtype=torch.bfloat16, device=dev).expand(batch, length, channels)
    D = torch.ones(channels, device=dev, requires_grad=True)
    lengths = torch.tensor(([length, length - 1, 0, 513, 512, 1, 9000] * 2)[:batch] if with_lengths else [length] * batch)
    grad = torch.full((batch, length, channels), E, dtype=torch.bfloat16, device=dev)
    grad[:, -1] = 1.0   # (the walk back begins there)
    out = S.state_space_scan(x, zero, torch.zeros(channels, 1, device=dev), bc, bc, D=D, softplus=False, lengths=lengths.to(dev, torch.int32))
    got, = torch.autograd.grad(out, D, grad)
    full = int((lengths == length).sum())
    check(got, full + (int(lengths.sum()) - full) * E, "D")


def test_shared_gradients_of_many_channels(dev):
    """dB and dC are sums over the channels: 64 in a workgroup, in float32 (8 roundings), and 4096 such blocks."""
    channels = 64 * 4096
    x = ones(dev, torch.bfloat16, 1, 1, channels)
    B, C = torch.ones(1, 1, 1, 1, device=dev, requires_grad=True), torch.ones(1, 1, 1, 1, device=dev, requires_grad=True)
    grad = torch.zeros(1, 1, channels, dtype=torch.bfloat16, device=dev)
    grad[..., ::64] = E
    grad[..., 0] = 1.0
    out = S.state_space_scan(x, x, torch.zeros(channels, 1, device=dev), B, C, softplus=False)
    for name, g in zip("BC", torch.autograd.grad(out, (B, C), grad)):
        check(g, 1 + 4095 * E, name, 10)
