"""What the sequence and gradient operators decide on the host (no GPU needed)."""

import pytest
import torch
from torch.autograd import forward_ad

from isaaclab_amd.utils import gradients as G
from isaaclab_amd.utils import sequence as S


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
