"""Global gradient norm and clipping on ``ilx_gradient_norm`` (include/isaaclab_amd_sequence.h): the end of a training step.

No counterpart in the reference, whose RL libraries call torch.  All tensors, of any mix of float32, bfloat16 and float16, are
reduced in one launch per 223 tensors and scaled in place in another; nothing is read back to the host.  No derivative goes
through the norm or the scaling (forward mode is refused).  Squares are added in 64 bits in a fixed order, so their sum
neither overflows nor depends on scheduling: replicas with equal gradients clip alike.
"""

from __future__ import annotations

import contextlib
import math
import operator
from array import array
from collections.abc import Iterable
from ctypes import c_float, c_int32, c_int64

import torch

from .. import _abi
from .sequence import _DTYPES, _current_device, _keep, _no_tangents, _written

_norm = _abi._sig("ilx_gradient_norm", _abi.P, _abi.P, _abi.P, c_int32, c_int32, c_int32, c_float, _abi.P, _abi.P, c_int64, _abi.P)
_T, _dtype, _KIND = torch.Tensor, operator.attrgetter("dtype"), _DTYPES.get
_WORKSPACE = 4096   # floats, what ilx_gradient_norm_workspace says for any list


def _is_dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one block of memory, in any order of the dimensions."""
    return t.is_contiguous() or torch.empty_like(t, device="meta").stride() == t.stride()


def _call(gradients: Iterable[torch.Tensor | None], norm_type: float, clip: bool, max_norm: float) -> torch.Tensor:
    if norm_type not in (2, 2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if isinstance(gradients, torch.Tensor):
        gradients = [gradients]
    tensors = [g for g in gradients if g is not None]
    if not tensors:
        raise ValueError("no gradients")
    _no_tangents(tensors)
    first = tensors[0]
    if not first.is_cuda:
        raise _abi.IlxError("isaaclab_amd kernels need GPU tensors (got a CPU tensor); there is no CPU fallback")
    index = first.get_device()
    kinds = list(map(_KIND, map(_dtype, tensors)))   # (map: a training step may have hundreds of tensors)
    if None in kinds or set(map(_T.get_device, tensors)) != {index} or not all(map(_T.is_contiguous, tensors)):
        for i, g in enumerate(tensors):
            if g.get_device() != index:
                raise ValueError(f"gradient {i} is on {g.device}, the first on {first.device}")
            if g.dtype not in _DTYPES:
                raise ValueError(f"gradient {i} is {g.dtype}: float32, bfloat16 or float16 expected")
            if g.layout != torch.strided or not _is_dense(g):
                raise ValueError(f"gradient {i} is not dense: strides {g.stride() if g.layout == torch.strided else g.layout} of shape {tuple(g.shape)}")
    pointers, sizes, dtypes = array("q", map(_T.data_ptr, tensors)), array("q", map(_T.numel, tensors)), array("i", kinds)
    norm = _abi.keep(torch.empty((), device=first.device))
    workspace = _abi.keep(torch.empty(_WORKSPACE, device=first.device))
    _keep(*tensors)
    with contextlib.nullcontext() if index == _current_device() else torch.cuda.device(index):
        status = _norm(pointers.buffer_info()[0], sizes.buffer_info()[0], dtypes.buffer_info()[0], len(tensors), int(norm_type == math.inf),
                       int(clip), max_norm, norm.data_ptr(), workspace.data_ptr(), _WORKSPACE, _abi.stream())
    _abi.check(status, "ilx_gradient_norm")
    if clip:
        _written(tensors)
    return norm


def gradient_norm(gradients: Iterable[torch.Tensor | None], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all ``gradients`` as one vector, a float32 scalar on their device.  ``None`` entries (parameters without a
    gradient) are left out; ``norm_type`` is 2 or ``math.inf``."""
    return _call(gradients, norm_type, False, 0.0)


def clip_gradient_norm(gradients: Iterable[torch.Tensor | None], max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """Scale ``gradients`` in place by ``min(1, max_norm / (norm + 1e-6))`` and return the norm they had.

    A norm that is not finite scales as the formula says (infinity: finite gradients become 0, NaN: all become NaN).
    Tensors must be dense and share no memory; a list of ``[p.grad for p in parameters]`` is what is meant."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return _call(gradients, norm_type, True, max_norm)
