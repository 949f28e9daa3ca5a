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
