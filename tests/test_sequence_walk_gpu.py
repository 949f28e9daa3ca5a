"""GPU: the operators where a wave (forward) or a workgroup (backward) takes several sequences or parts one after the other.

A chip of 256 CUs is full with 4096 waves and 1536 workgroups; from there on each walks more than one item: the next sequence's rows
are read while the last one's state and the zeros behind its end are written, its state and its gradient are taken up anew, and
empty sequences are crossed.  Oracle and bounds are those of tests/test_sequence_gpu.py."""

import ctypes

import pytest
import test_sequence_gpu as base
import torch

from isaaclab_amd.utils import sequence as S

pytestmark = pytest.mark.gpu

F32, BF16, F16 = 0, 1, 2
CASES = [  # batch, length, channels, states, groups, dtype, shared in float32, gate, softplus, starts, lengths, state, time major
    (5003, 9, 20, 5, 1, F32, False, True, True, True, True, True, True),       # two forward, four backward, the last one short
    (5003, 9, 20, 16, 1, BF16, False, True, True, False, True, True, False),
    (2111, 12, 130, 16, 2, BF16, False, True, True, True, True, True, True),   # 65 channels to a group: two blocks, one of one channel
    (2111, 12, 66, 4, 2, F32, False, False, True, True, False, True, False),
    (6001, 5, 12, 32, 1, F32, False, True, False, True, True, True, True),
    (4500, 17, 24, 7, 1, F16, True, True, True, False, True, True, True),
    (8200, 1, 40, 8, 2, F16, False, False, True, True, False, True, False),    # one row each
    (8200, 2, 10, 16, 1, F32, False, True, True, False, True, False, False),
    (500, 130, 20, 5, 1, F32, False, True, True, True, True, True, True),      # divided: six parts each, two to a workgroup backward
    (700, 200, 9, 16, 1, BF16, False, True, True, False, True, True, False),
]


@pytest.mark.parametrize("case", CASES)
def test_scan_and_its_gradients(dev, case):
    batch, length, channels, states, groups = case[:5]
    # so many items come to a workgroup of the backward pass: the workspace holds a row of partial sums each
    desc = S.StateSpaceDesc(batch=batch, length=length, channels=channels, states=states, groups=groups)
    forward, both = ctypes.c_int64(), ctypes.c_int64()
    assert S._scan_workspace(ctypes.byref(desc), 0, ctypes.byref(forward)) == 0 and S._scan_workspace(ctypes.byref(desc), 1, ctypes.byref(both)) == 0
    blocks = -(-(channels // groups) // 64)
    padded = 8 * (1 if states <= 4 else 2 if states <= 8 else 4 if states <= 16 else 8)
    rows = (both.value - forward.value - blocks * batch * length * groups * padded) // ((states + 2) * channels)
    items = batch if forward.value == 0 else forward.value // ((states + 1) * channels)
    assert items > rows > 0
    base.test_scan_and_its_gradients(dev, *case)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_empty_sequences_in_between(dev, dtype):
    """Every third sequence empty, every third whole, every third cut: results and gradients of each are those of the sequence alone
    among a few (whose path the oracle checks), states pass through the empty ones, and nothing behind an end is read."""
    batch, length, channels, states = 4803, 11, 24, 8
    gen = torch.Generator().manual_seed(3)
    v = {k: t.to(dev) for k, t in base.scan_inputs(gen, batch, length, channels, states, 1, dtype, False, True, True, True, True).items()}
    lengths = torch.tensor([0, length, 5] * (batch // 3), device=dev, dtype=torch.int32)
    inside = (torch.arange(length, device=dev) < lengths[:, None])
    for k in ("x", "delta", "gate", "B", "C"):
        v[k][~inside] = float("nan")
    grad, grad_last = torch.randn(batch, length, channels, device=dev).to(dtype), torch.randn(batch, states, channels, device=dev)
    names = ("x", "delta", "B", "C", "gate", "state")

    def run(pick):
        w = {k: t[pick].contiguous() if k in names else t for k, t in v.items()}
        leaves = {k: w[k].detach().requires_grad_(True) for k in names}
        out, last = base.run_scan({**w, **leaves}, lengths=lengths[pick])
        return [out, last, *torch.autograd.grad([out, last], list(leaves.values()), [grad[pick], grad_last[pick]])]

    every = run(torch.arange(batch, device=dev))
    for i in (0, 1, 2, 4, 1500, 2401, 2402, 2403, 4500, 4801, 4802):
        for name, a, b in zip(("out", "last", *names), every, run(torch.tensor([i], device=dev))):
            assert torch.equal(a[i:i + 1], b), (i, name)
    out, last, *grads = every
    assert not out[~inside].any() and torch.equal(last[::3], v["state"][::3]) and torch.equal(grads[5][::3], grad_last[::3])
    assert all(not g[~inside].any() and g.isfinite().all() for g in grads[:5])


@pytest.mark.parametrize("case", [   # batch, length, channels, width, dtype, silu, starts, lengths, state, time major
    (5003, 5, 70, 4, F32, True, True, True, True, True),      # three sequences to a thread of the backward pass
    (9001, 3, 33, 2, F16, False, True, True, True, False),
    (40, 1300, 130, 5, BF16, True, True, True, True, True),   # two segments
])
def test_convolution_and_its_gradients(dev, case):
    base.test_convolution_and_its_gradients(dev, *case)
