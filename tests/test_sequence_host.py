"""What the sequence and gradient operators decide on the host (no GPU needed)."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from isaaclab_amd import _abi
from isaaclab_amd.utils import gradients as G
from isaaclab_amd.utils import sequence as S
from isaaclab_amd.utils.command_list import CommandList
from oracle import sequence as O


def test_forward_mode_is_refused():
    """A dual tensor does not require gradients; passed to a kernel its tangent would be gone."""
    x = torch.randn(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        for call in (lambda: S._needs_gradients((x, None, dual)), lambda: S._no_gradients("a step", (dual, x)), lambda: G.gradient_norm([x, dual]),
                     lambda: G.clip_gradient_norm([dual], 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert not S._needs_gradients((x, None))   # operands without a tangent pass inside a level
    assert not S._needs_gradients((x,))


def test_overlap_of_rows_and_a_dense_block():
    """Against the sets of elements that the two touch."""
    memory = torch.zeros(400)
    seen = set()
    for at in range(0, 60, 7):
        dense = memory[100:100 + 3 * 5 * 4].view(3, 5, 4)
        for batch, step, width in ((1, 1, 4), (3, 4, 4), (3, 11, 4), (2, 150, 30), (4, 70, 9), (2, 0, 5)):
            for offset in (0, 60, 95 + at % 11, 100 + at, 155 + at % 9):
                rows = memory.as_strided((batch, width), (step, 1), offset)
                touched = {offset + b * step + c for b in range(batch) for c in range(width)}
                want = bool(touched & set(range(100, 160)))
                assert S._overlap(rows, dense) == want, (batch, step, width, offset)
                seen.add(want)
    assert seen == {True, False}
    assert not S._overlap(memory[:0].view(0, 4), memory) and not S._overlap(memory.view(20, 20), memory[:0])


def test_rows_are_counted_in_32_bits():
    """Where the last part of a divided sequence ends stays below 2^31 for every accepted length; longer ones are refused."""
    most = 2 ** 31 - 4097
    need = ctypes.c_int64()

    def parts_of(length, batch, channels):
        desc = S.StateSpaceDesc(batch=batch, length=length, channels=channels, states=1, groups=1)
        status = S._scan_workspace(ctypes.byref(desc), 0, ctypes.byref(need))
        return status, need.value // (2 * batch * channels)   # a state and a decay per part and channel

    for batch, channels in ((1, 1), (1, 64), (3, 64), (7, 640), (250, 256)):
        for length in (most, most - 1, most - 57, 2 ** 31 - 2 ** 23, 2 ** 30 + 1, 2 ** 24 + 9):
            status, parts = parts_of(length, batch, channels)
            assert status == 0 and 1 < parts <= 256
            rows = -(-(-(-length // parts)) // 8) * 8   # the fewest rows, a multiple of 8, that make as many parts ...
            while -(-length // rows) > parts:
                rows += 8
            assert parts * rows < 2 ** 31, (batch, channels, length, parts)   # ... and its last part ends here
        assert parts_of(most + 1, batch, channels)[0] == -2 and b"too large" in _abi.lib.ilx_last_error()


def test_launches_of_a_gradient_list():
    """Two launches (one and one more for the norm alone) for as many tensors as fit a kernel's arguments; empty tensors take no place."""
    most = 223

    def launches(sizes, clip):
        n, at = len(sizes), 0x100000
        pointers = [at := at + 0x10000 for _ in sizes]
        commands = CommandList()
        with commands.record():   # (what the call answers without a device does not matter)
            G._norm((ctypes.c_void_p * n)(*pointers), (ctypes.c_int64 * n)(*sizes), (ctypes.c_int32 * n)(), n, 0, clip, 1.0, 0x1000, 0x2000, 4096, None)
        return len(commands)

    for count, tables in ((1, 1), (16, 1), (200, 1), (201, 1), (most, 1), (most + 1, 2), (2 * most, 2), (2 * most + 1, 3)):
        assert launches([7] * count, 1) == 2 * tables and launches([7] * count, 0) == tables + 1, count
        assert launches([0, 7] * count, 1) == 2 * tables, count
    assert launches([0], 1) == 2


def test_the_oracle_s_step_size():
    """log(1 + e^x) and its slope 1 / (1 + e^-x), at zero too."""
    x = torch.tensor([0.0, 1e-300, -1e-12, 0.5, -0.5, 3.0, -3.0, 30.0, -30.0, 700.0, -700.0], dtype=torch.float64, requires_grad=True)
    value = O._softplus(x)
    slope, = torch.autograd.grad(value.sum(), x)
    want = torch.where(x > 0, x + torch.log1p(torch.exp(-x.abs())), torch.log1p(torch.exp(x)))
    torch.testing.assert_close(value, want, rtol=1e-15, atol=0)
    torch.testing.assert_close(slope, 1 / (1 + torch.exp(-x.detach())), rtol=1e-13, atol=0)
