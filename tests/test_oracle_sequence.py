"""The sequence oracle against differences, and against itself cut in two; the refusals of the C calls (no GPU needed)."""

import ctypes

import pytest
import torch

from isaaclab_amd import _abi
from isaaclab_amd.utils import gradients as G
from isaaclab_amd.utils import sequence as S
from oracle import sequence as O

EINVAL, ESHAPE = -1, -2
FAKE = 0x1000


def leaf(*shape, scale=1.0):
    return (torch.randn(*shape, dtype=torch.float64) * scale).requires_grad_(True)


def test_short_convolution_gradients_against_differences():
    torch.manual_seed(0)
    starts = torch.tensor([[0, 0, 1, 0, 0], [1, 0, 0, 0, 1]])
    lengths = torch.tensor([5, 3])
    f = lambda x, w, b, s: O.short_convolution(x, w, b, True, s, starts, lengths)  # noqa: E731
    assert torch.autograd.gradcheck(f, (leaf(2, 5, 3), leaf(3, 4), leaf(3), leaf(2, 3, 3)))


def test_state_space_gradients_against_differences():
    torch.manual_seed(1)
    starts = torch.tensor([[0, 0, 1, 0, 0], [1, 0, 0, 0, 1]])
    lengths = torch.tensor([5, 3])
    f = lambda x, d, A, B, C, D, z, b, s: O.state_space_scan(x, d, A, B, C, D, z, b, True, s, starts, lengths)  # noqa: E731
    args = (leaf(2, 5, 4), leaf(2, 5, 4), leaf(4, 3), leaf(2, 5, 2, 3), leaf(2, 5, 2, 3), leaf(4), leaf(2, 5, 4), leaf(4), leaf(2, 3, 4))
    assert torch.autograd.gradcheck(f, args)


def test_a_sequence_cut_in_two_is_the_whole():
    torch.manual_seed(2)
    x, w, b, s = leaf(2, 7, 3), leaf(3, 4), leaf(3), leaf(2, 3, 3)
    out, last = O.short_convolution(x, w, b, True, s)
    o1, l1 = O.short_convolution(x[:, :2], w, b, True, s)
    o2, l2 = O.short_convolution(x[:, 2:], w, b, True, l1)
    assert torch.equal(torch.cat([o1, o2], 1), out) and torch.equal(l2, last)


def fails(status, code, needle):
    msg = _abi.lib.ilx_last_error().decode()
    assert status == code and needle in msg, (status, msg)


def conv(**kw):
    d = dict(x=FAKE, weight=FAKE, out=FAKE, batch=2, length=4, channels=8, width=4, dtype=0)
    d.update(kw)
    return ctypes.byref(S.ShortConvDesc(**d))


def test_short_conv_refusals():
    fails(S._conv_forward(None, None), EINVAL, "NULL")
    fails(S._conv_forward(conv(x=None), None), EINVAL, "ilx_short_conv_forward: NULL operand")
    fails(S._conv_forward(conv(weight=None), None), EINVAL, "NULL operand")
    fails(S._conv_forward(conv(width=9), None), ESHAPE, "width 9")
    fails(S._conv_forward(conv(width=0), None), ESHAPE, "width 0")
    fails(S._conv_forward(conv(channels=0), None), EINVAL, "bad shape")
    fails(S._conv_forward(conv(length=-1), None), EINVAL, "bad shape")
    fails(S._conv_forward(conv(dtype=3), None), EINVAL, "unknown type 3")
    fails(S._conv_forward(conv(batch=1 << 30, length=1 << 20), None), ESHAPE, "too large")
    fails(S._conv_forward(conv(state=FAKE, last=FAKE), None), EINVAL, "same buffer")
    assert S._conv_forward(conv(batch=0, x=None, out=None), None) == 0
    fails(S._conv_backward(conv(grad_weight=FAKE), None), EINVAL, "ilx_short_conv_backward: NULL operand")
    grads = dict(grad_out=FAKE, grad_x=FAKE, grad_weight=FAKE)
    need = ctypes.c_int64()
    assert S._conv_workspace(conv(**grads), ctypes.byref(need)) == 0 and need.value > 0
    fails(S._conv_backward(conv(workspace=FAKE, workspace_floats=need.value - 1, **grads), None), EINVAL, "workspace")
    fails(S._conv_backward(conv(workspace_floats=need.value, **grads), None), EINVAL, "workspace")
    fails(S._conv_step(conv(), None), EINVAL, "ilx_short_conv_step: NULL operand")
    fails(S._conv_step(conv(state=FAKE, last=FAKE * 2), None), EINVAL, "in place")
    fails(S._conv_step(conv(state=FAKE, last=FAKE, lengths=FAKE), None), EINVAL, "lengths")


def scan(**kw):
    d = dict(x=FAKE, delta=FAKE, A=FAKE, B=FAKE, C=FAKE, out=FAKE, batch=2, length=4, channels=8, states=4, groups=1)
    d.update(kw)
    return ctypes.byref(S.StateSpaceDesc(**d))


def test_state_space_refusals():
    fails(S._scan_forward(None, None), EINVAL, "NULL")
    for name in ("x", "delta", "A", "B", "C", "out"):
        fails(S._scan_forward(scan(**{name: None}), None), EINVAL, "ilx_state_space_forward: NULL operand")
    fails(S._scan_forward(scan(states=33), None), ESHAPE, "33 states")
    fails(S._scan_forward(scan(states=0), None), ESHAPE, "0 states")
    fails(S._scan_forward(scan(groups=3), None), ESHAPE, "3 groups")
    fails(S._scan_forward(scan(groups=0), None), EINVAL, "0 groups")
    fails(S._scan_forward(scan(dtype=7), None), EINVAL, "unknown type 7")
    fails(S._scan_forward(scan(dtype=1, bc_dtype=2), None), EINVAL, "B and C of type 2")
    fails(S._scan_forward(scan(x_time=1 << 32), None), ESHAPE, "time stride")
    fails(S._scan_forward(scan(out_time=1 << 27), None), ESHAPE, "time stride")
    fails(S._scan_forward(scan(channels=(1 << 23) + 8), None), ESHAPE, "8388616 channels")
    fails(S._scan_forward(scan(length=2000, channels=64), None), EINVAL, "workspace")
    fails(S._scan_forward(scan(state=FAKE, last=FAKE), None), EINVAL, "same buffer")
    assert S._scan_forward(scan(batch=0, x=None), None) == 0
    grads = dict(grad_out=FAKE, grad_x=FAKE, grad_delta=FAKE, grad_A=FAKE, grad_B=FAKE, grad_C=FAKE, saved=FAKE)
    fails(S._scan_backward(scan(**dict(grads, saved=None)), None), EINVAL, "ilx_state_space_backward: NULL operand")
    fails(S._scan_backward(scan(gate=FAKE, **grads), None), EINVAL, "come together")
    need = ctypes.c_int64()
    assert S._scan_workspace(scan(**grads), 1, ctypes.byref(need)) == 0 and need.value > 0
    fails(S._scan_backward(scan(workspace=FAKE, workspace_floats=need.value - 1, **grads), None), EINVAL, "workspace")
    fails(S._scan_step(scan(), None), EINVAL, "ilx_state_space_step: NULL operand")
    fails(S._scan_step(scan(state=FAKE, last=2 * FAKE), None), EINVAL, "in place")


def test_gradient_norm_refusals():
    def call(pointers, sizes, dtypes, kind=0, clip=1, max_norm=1.0, norm=FAKE, workspace=FAKE, floats=4096, count=None):
        n = len(pointers)
        return G._norm((ctypes.c_void_p * n)(*pointers), (ctypes.c_int64 * n)(*sizes), (ctypes.c_int32 * n)(*dtypes), n if count is None else count, kind,
                       clip, max_norm, norm, workspace, floats, None)

    fails(call([FAKE], [4], [0], kind=2), EINVAL, "ilx_gradient_norm: unknown norm 2")
    fails(call([FAKE], [4], [0], norm=None), EINVAL, "norm is NULL")
    fails(call([FAKE], [4], [0], max_norm=-1.0), EINVAL, "max_norm")
    fails(call([FAKE], [4], [0], max_norm=float("nan")), EINVAL, "max_norm")
    fails(call([FAKE], [4], [0], floats=100), EINVAL, "workspace")
    fails(call([FAKE], [4], [0], workspace=FAKE + 4), EINVAL, "workspace")
    fails(call([None], [4], [0]), EINVAL, "tensor 0 is NULL")
    fails(call([FAKE], [-4], [0]), EINVAL, "tensor 0")
    fails(call([FAKE], [4], [5]), EINVAL, "type 5")
    fails(call([FAKE + 2], [4], [0]), EINVAL, "aligned")
    fails(call([FAKE, FAKE], [4, 4], [0, 0]), EINVAL, "tensors 0 and 1 share memory")
    fails(call([2 * FAKE, FAKE], [4, FAKE // 4 + 1], [0, 0]), EINVAL, "share memory")
    fails(call([FAKE], [4], [0], count=-1), EINVAL, "bad tensor list")


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(1, 2, 4), torch.zeros(4, 4)
    calls = [lambda: S.short_convolution(x, w), lambda: S.short_convolution_step(x[:, 0], torch.zeros(1, 3, 4), w),
             lambda: S.state_space_scan(x, x, w, x, x), lambda: S.state_space_step(x[:, 0], x[:, 0], torch.zeros(1, 4, 4), w, x[:, 0], x[:, 0]),
             lambda: G.clip_gradient_norm([w], 1.0), lambda: G.gradient_norm([w])]
    for call in calls:
        with pytest.raises(_abi.IlxError, match="GPU"):
            call()
