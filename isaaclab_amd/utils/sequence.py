"""The memory of a recurrent policy or actuator over time: a short causal convolution and a selective state space recurrence
on the HIP kernels ``ilx_short_conv_*`` / ``ilx_state_space_*`` (include/isaaclab_amd_sequence.h).

No counterpart in the reference, whose recurrent models are torch modules of the RL libraries.  Like the modifiers and the
LSTM actuator each operator keeps a state per environment, and it comes in two forms that agree:

* over a sequence (``short_convolution``, ``state_space_scan``): a rollout of all environments or a recording at once, with
  gradients for training;
* one environment step (``short_convolution_step``, ``state_space_step``): one row per environment on a carried state, which is
  updated in place; no gradients.

    out, last = state_space_scan(x, delta, A, B, C, D=D, gate=z, state=state, starts=dones_before, return_state=True)
    ...
    out = state_space_step(x, delta, last, A, B, C, D=D, gate=z, starts=env.reset_buf)

Activations are (batch, length, channels) in float32, bfloat16 or float16, with any batch and time strides: a time-major
rollout buffer goes in as ``buffer.transpose(0, 1)``, and the output has its layout.  Parameters and states are float32, and
everything is computed in float32.  ``starts`` (batch, length) marks the rows on which an episode begins: nothing from before
such a row, the carried state included, reaches it.  ``lengths`` (batch) says where a padded sequence ends: rows behind are
not read, their outputs and gradients are zero, and the state skips them.

As everywhere in this package there is no CPU fallback.  Inside ``CommandList.record`` the calls are recorded, and the list keeps
their operands and the buffers they allocate; a call whose operands need gradients is refused there (its backward pass runs on
another thread).  Forward-mode differentiation is refused, and so are second derivatives.
"""

from __future__ import annotations

import ctypes
from ctypes import c_int32, c_int64, c_void_p

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _abi

MAX_WIDTH = 8
MAX_STATES = 32
_BLOCK = 8   # ILX_SCAN_BLOCK
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class ShortConvDesc(ctypes.Structure):
    """Mirror of ``ilx_short_conv`` (include/isaaclab_amd_sequence.h)."""

    _fields_ = [
        ("x", c_void_p), ("x_batch", c_int64), ("x_time", c_int64), ("weight", c_void_p), ("bias", c_void_p), ("state", c_void_p),
        ("starts", c_void_p), ("starts_batch", c_int64), ("starts_time", c_int64), ("lengths", c_void_p),
        ("out", c_void_p), ("out_batch", c_int64), ("out_time", c_int64), ("last", c_void_p), ("batch", c_int64), ("length", c_int64),
        ("channels", c_int32), ("width", c_int32), ("dtype", c_int32), ("silu", c_int32),
        ("grad_out", c_void_p), ("grad_out_batch", c_int64), ("grad_out_time", c_int64), ("grad_last", c_void_p),
        ("grad_x", c_void_p), ("grad_x_batch", c_int64), ("grad_x_time", c_int64), ("grad_weight", c_void_p), ("grad_bias", c_void_p),
        ("grad_state", c_void_p), ("workspace", c_void_p), ("workspace_floats", c_int64),
    ]


class StateSpaceDesc(ctypes.Structure):
    """Mirror of ``ilx_state_space`` (include/isaaclab_amd_sequence.h)."""

    _fields_ = [
        ("x", c_void_p), ("x_batch", c_int64), ("x_time", c_int64), ("delta", c_void_p), ("delta_batch", c_int64), ("delta_time", c_int64),
        ("gate", c_void_p), ("gate_batch", c_int64), ("gate_time", c_int64), ("A", c_void_p),
        ("B", c_void_p), ("B_batch", c_int64), ("B_time", c_int64), ("C", c_void_p), ("C_batch", c_int64), ("C_time", c_int64),
        ("D", c_void_p), ("delta_bias", c_void_p), ("state", c_void_p), ("starts", c_void_p), ("starts_batch", c_int64),
        ("starts_time", c_int64), ("lengths", c_void_p), ("out", c_void_p), ("out_batch", c_int64), ("out_time", c_int64),
        ("last", c_void_p), ("saved", c_void_p), ("batch", c_int64), ("length", c_int64), ("channels", c_int32), ("states", c_int32),
        ("groups", c_int32), ("dtype", c_int32), ("bc_dtype", c_int32), ("softplus", c_int32),
        ("grad_out", c_void_p), ("grad_out_batch", c_int64), ("grad_out_time", c_int64), ("grad_last", c_void_p),
        ("grad_x", c_void_p), ("grad_delta", c_void_p), ("grad_gate", c_void_p), ("grad_batch", c_int64), ("grad_time", c_int64),
        ("grad_A", c_void_p), ("grad_B", c_void_p), ("grad_C", c_void_p), ("grad_D", c_void_p), ("grad_delta_bias", c_void_p),
        ("grad_state", c_void_p), ("workspace", c_void_p), ("workspace_floats", c_int64),
    ]


_P = c_void_p
_conv_forward = _abi._sig("ilx_short_conv_forward", _P, _P)
_conv_workspace = _abi._sig("ilx_short_conv_workspace", _P, _P)
_conv_backward = _abi._sig("ilx_short_conv_backward", _P, _P)
_conv_step = _abi._sig("ilx_short_conv_step", _P, _P)
_scan_forward = _abi._sig("ilx_state_space_forward", _P, _P)
_scan_workspace = _abi._sig("ilx_state_space_workspace", _P, c_int32, _P)
_scan_backward = _abi._sig("ilx_state_space_backward", _P, _P)
_scan_step = _abi._sig("ilx_state_space_step", _P, _P)


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)   # (without the lazy-initialisation check)


def _launch(fn, desc, what: str, index: int):
    """One call on the tensors' device and its current stream."""
    if index == _current_device():
        _abi.check(fn(ctypes.byref(desc), _abi.stream()), what)
    else:
        with torch.cuda.device(index):
            _abi.check(fn(ctypes.byref(desc), _abi.stream()), what)


def _p(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _copy(t: torch.Tensor, name: str, **how) -> torch.Tensor:
    """A dense copy (``how``: in another type).  A recorded call would go on reading the values of the recording."""
    if _abi.recording():
        raise _abi.IlxError(f"{name} would be copied before the call, which a command list does not record: pass it dense, and B and C in one type")
    return t.to(**how).contiguous()


def _on(t: torch.Tensor, name: str, index: int):
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the activations on cuda:{index}")


def _check_activation(t: torch.Tensor, name: str, like: torch.Tensor, index: int) -> torch.Tensor:
    """``t`` with unit channel stride (copied only if it has another)."""
    if t.shape != like.shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(like.shape)}")
    if t.dtype is not like.dtype:
        raise ValueError(f"{name} is {t.dtype} beside {like.dtype} activations")
    _on(t, name, index)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else _copy(t, name)


def _check_parameter(t: torch.Tensor | None, name: str, shape: tuple, index: int) -> torch.Tensor | None:
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if t.dtype is not torch.float32:
        raise ValueError(f"{name} is {t.dtype}: parameters and states are float32")
    _on(t, name, index)
    return t if t.is_contiguous() else _copy(t, name)


def _check_x(x: torch.Tensor, dims: int) -> tuple[torch.Tensor, int]:
    """x with unit channel stride, and its device."""
    if not x.is_cuda:
        raise _abi.IlxError("isaaclab_amd kernels need GPU tensors (got a CPU tensor); there is no CPU fallback")
    if x.dim() != dims:
        raise ValueError(f"x has shape {tuple(x.shape)}, expected {'(batch, length, channels)' if dims == 3 else '(batch, channels)'}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"activations are float32, bfloat16 or float16, got {x.dtype}")
    if x.shape[-1] == 0:
        raise ValueError("x has no channels")
    return (x if x.stride(-1) == 1 or x.shape[-1] == 1 else _copy(x, "x")), x.get_device()


def _check_starts(starts: torch.Tensor | None, shape: tuple, index: int) -> torch.Tensor | None:
    if starts is not None:
        if starts.shape != shape or starts.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"starts is {starts.dtype} {tuple(starts.shape)}, expected bool {shape}")
        _on(starts, "starts", index)
    return starts


def _check_lengths(lengths: torch.Tensor | None, batch: int, length: int, index: int) -> torch.Tensor | None:
    if lengths is None:
        return None
    if lengths.shape != (batch,) or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"lengths is {lengths.dtype} {tuple(lengths.shape)}, expected int32 or int64 {(batch,)}")
    _on(lengths, "lengths", index)
    if lengths.dtype is torch.int64 and not _abi.recording():
        lengths = lengths.clamp(0, length)   # (ahead of the narrowing, which would wrap)
    return lengths if lengths.dtype is torch.int32 and lengths.is_contiguous() else _copy(lengths, "lengths", dtype=torch.int32)


def _check_state(state: torch.Tensor, shape: tuple, index: int):
    """A state that is updated in place: it cannot be a copy."""
    if not isinstance(state, torch.Tensor):
        raise ValueError("a step needs its carried state (zeros for a new sequence)")
    if not state.is_contiguous():
        raise ValueError("state is updated in place and must be contiguous")
    _check_parameter(state, "state", shape, index)


def _wants_gradients(tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tangents(tensors):
    """A dual tensor of forward-mode differentiation does not say ``requires_grad``: its tangent would be lost without a word."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("forward-mode differentiation is not supported: an operand carries a tangent")


def _no_gradients(what: str, tensors):
    _no_tangents(tensors)
    if _wants_gradients(tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad(), or use the form over sequences")


def _needs_gradients(tensors) -> bool:
    _no_tangents(tensors)
    if not _wants_gradients(tensors):
        return False
    if _abi.recording():
        raise _abi.IlxError("a call that needs gradients cannot be recorded in a command list (its backward pass runs on another thread)")
    return True


def _overlap(rows: torch.Tensor, dense: torch.Tensor) -> bool:
    """Whether a row of ``rows`` (unit channel stride) touches the memory of ``dense``."""
    if rows.numel() == 0 or dense.numel() == 0:
        return False
    size = rows.element_size()
    begin, step, width = rows.data_ptr(), rows.stride(0) * size, rows.shape[1] * size
    lo, hi = dense.data_ptr(), dense.data_ptr() + dense.numel() * dense.element_size()
    first = 0 if begin + width > lo or step == 0 else (lo - begin - width) // step + 1   # the first row that ends behind lo
    return first < rows.shape[0] and begin + first * step < hi and begin + first * step + width > lo


def _check_out(out: torch.Tensor | None, x: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    if out is None:
        return _empty_like(x)
    if out.shape != x.shape or out.dtype is not x.dtype or out.device != x.device or (out.stride(-1) != 1 and out.shape[-1] != 1):
        raise ValueError(f"out must be like x ({tuple(x.shape)}, {x.dtype}) with unit channel stride")
    if out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError(f"out's rows overlap (strides {out.stride()})")
    if _overlap(out, state):
        raise ValueError("out and state share memory, and both are written")
    return out


def _empty_like(x: torch.Tensor) -> torch.Tensor:
    """Dense, in x's order of batch and time; where x is a view whose rows overlap (a sliding window), in the plain order."""
    out = torch.empty_like(x)
    return out if out.stride(-1) == 1 or out.shape[-1] == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _keep(*tensors):
    """What a recorded call reads or writes stays alive with its list."""
    if _abi.recording():
        for t in tensors:
            _abi.keep(t)


def _written(tensors):
    """Autograd sees the in-place update: a backward pass that needs a value from before it fails loudly."""
    if any(map(torch.Tensor.is_inference, tensors)):
        tensors = [t for t in tensors if not t.is_inference()]
    torch.autograd.graph.increment_version(tensors)


def _places(tensors) -> list:
    return [None if t is None else (t.data_ptr(), t.stride()) for t in tensors]


def _once(backward):
    """A backward pass that cannot be differentiated again (without ``create_graph`` there is nothing to guard) nor recorded."""
    guarded = once_differentiable(backward)

    def either(ctx, *grads):
        if _abi.recording():   # (autograd on the calling thread: torch.autograd.set_multithreading_enabled(False))
            raise _abi.IlxError("a backward pass cannot be recorded in a command list")
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return either


# ---- short convolution ----------------------------------------------------------------------------------------------
def _silu(activation) -> int:
    if activation not in (None, "silu"):
        raise ValueError(f"unsupported activation '{activation}', expected None or 'silu'")
    return int(activation == "silu")


def _conv_desc(x, weight, bias, state, starts, lengths, silu) -> ShortConvDesc:
    batch, length, channels = x.shape
    x_batch, x_time, _ = x.stride()
    starts_batch, starts_time = starts.stride() if starts is not None else (0, 0)
    # (in the order of the fields)
    return ShortConvDesc(
        x.data_ptr(), x_batch, x_time, weight.data_ptr(), _p(bias), _p(state), _p(starts), starts_batch, starts_time, _p(lengths),
        None, 0, 0, None, batch, length, channels, weight.shape[1], _DTYPES[x.dtype], silu)


def _conv_call(x, weight, bias, state, starts, lengths, silu, want_last):
    desc = _conv_desc(x, weight, bias, state, starts, lengths, silu)
    out = _empty_like(x)
    last = torch.empty(x.shape[0], weight.shape[1] - 1, x.shape[2], device=x.device) if want_last else None
    _keep(x, weight, bias, state, starts, lengths, out, last)
    desc.out, desc.last = out.data_ptr(), _p(last)
    desc.out_batch, desc.out_time, _ = out.stride()
    _launch(_conv_forward, desc, "ilx_short_conv_forward", x.get_device())
    return out, last, desc


class _ShortConvolution(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, starts, lengths, silu, want_last):
        ctx.set_materialize_grads(False)
        saved = (x, weight, bias, state, starts, lengths)
        ctx.save_for_backward(*saved)
        ctx.places = _places(saved)
        out, last, ctx.desc = _conv_call(x, weight, bias, state, starts, lengths, silu, want_last)
        return out, last

    @staticmethod
    @_once
    def backward(ctx, grad_out, grad_last):
        x, weight, bias, state, starts, lengths = saved = ctx.saved_tensors
        d = ctx.desc
        if _places(saved) != ctx.places:   # (hooks may pack saved tensors and unpack them elsewhere)
            d = _conv_desc(x, weight, bias, state, starts, lengths, d.silu)
        index = x.get_device()
        grad_out = torch.zeros_like(x) if grad_out is None else _check_activation(grad_out, "the output's gradient", x, index)
        grad_last = None if grad_last is None else grad_last.contiguous()
        grad_x, grad_weight = _empty_like(x), torch.empty_like(weight)
        grad_bias = None if bias is None else torch.empty_like(bias)
        grad_state = torch.empty_like(state) if state is not None and ctx.needs_input_grad[3] else None
        d.grad_out, d.grad_last, d.grad_x = grad_out.data_ptr(), _p(grad_last), grad_x.data_ptr()
        d.grad_out_batch, d.grad_out_time, _ = grad_out.stride()
        d.grad_x_batch, d.grad_x_time, _ = grad_x.stride()
        d.grad_weight, d.grad_bias, d.grad_state = grad_weight.data_ptr(), _p(grad_bias), _p(grad_state)
        need = c_int64()
        _abi.check(_conv_workspace(ctypes.byref(d), ctypes.byref(need)), "ilx_short_conv_workspace")
        workspace = torch.empty(need.value, device=x.device)
        d.workspace, d.workspace_floats = workspace.data_ptr(), need.value
        _launch(_conv_backward, d, "ilx_short_conv_backward", index)
        return grad_x, grad_weight, grad_bias, grad_state, None, None, None, None


def _check_filter(weight: torch.Tensor, bias, channels: int, index: int):
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_WIDTH:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, expected (channels, width) with a width of 1..{MAX_WIDTH}")
    return _check_parameter(weight, "weight", (channels, weight.shape[1]), index), _check_parameter(bias, "bias", (channels,), index)


def short_convolution(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
                      state: torch.Tensor | None = None, starts: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                      return_state: bool = False):
    """Causal convolution over time, one filter per channel: ``out[b, t] = act(bias + sum_j weight[:, W - 1 - j] * x[b, t - j])``.

    ``x`` (batch, length, channels), ``weight`` (channels, W) with W up to 8, ``activation`` None or ``"silu"``.  ``state``
    (batch, W - 1, channels) holds the rows ahead of the first, oldest first (zeros if None).  With ``return_state`` the
    result is ``(out, last)``, ``last`` being the state ahead of the next row.  Differentiable in ``x``, ``weight``,
    ``bias`` and ``state``."""
    x, index = _check_x(x, 3)
    batch, length, channels = x.shape
    silu = _silu(activation)
    weight, bias = _check_filter(weight, bias, channels, index)
    state = _check_parameter(state, "state", (batch, weight.shape[1] - 1, channels), index)
    starts = _check_starts(starts, (batch, length), index)
    lengths = _check_lengths(lengths, batch, length, index)
    if _needs_gradients((x, weight, bias, state)):
        out, last = _ShortConvolution.apply(x, weight, bias, state, starts, lengths, silu, return_state)
    else:
        out, last, _ = _conv_call(x, weight, bias, state, starts, lengths, silu, return_state)
    return (out, last) if return_state else out


def short_convolution_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                           activation: str | None = None, starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One row of :func:`short_convolution` per sequence: ``x`` (batch, channels), ``state`` (batch, W - 1, channels) updated in
    place, ``starts`` (batch) the environments whose episode begins with this row.  ``out`` may name the
    result's buffer, ``x`` itself for one, and shares memory with no other operand."""
    x, index = _check_x(x, 2)
    _no_gradients("short_convolution_step", (x, weight, bias, state, out))
    batch, channels = x.shape
    silu = _silu(activation)
    weight, bias = _check_filter(weight, bias, channels, index)
    width = weight.shape[1]
    _check_state(state, (batch, width - 1, channels), index)
    starts = _check_starts(starts, (batch,), index)
    written = (state,) if out is None else (state, out)
    out = _check_out(out, x, state)
    _keep(x, weight, bias, state, starts, out)
    at = state.data_ptr()
    desc = ShortConvDesc(
        x.data_ptr(), x.stride(0), 0, weight.data_ptr(), _p(bias), at, _p(starts), starts.stride(0) if starts is not None else 0, 0, None,
        out.data_ptr(), out.stride(0), 0, at, batch, 1, channels, width, _DTYPES[x.dtype], silu)
    _launch(_conv_step, desc, "ilx_short_conv_step", index)
    _written(written)
    return out


# ---- state space recurrence -------------------------------------------------------------------------------------------
def _shared(t: torch.Tensor, name: str, like: torch.Tensor, index: int) -> torch.Tensor:
    """B or C as (*lead, groups, states), dense over the last two: in the activations' type or float32."""
    lead = like.shape[:-1]
    if t.dim() == len(lead) + 1:
        t = t.unsqueeze(-2)
    if t.dim() != len(lead) + 2 or t.shape[:-2] != lead:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(lead)} + (groups, states) or (states,)")
    if t.dtype is not like.dtype and t.dtype is not torch.float32:
        raise ValueError(f"{name} is {t.dtype} beside {like.dtype} activations")
    _on(t, name, index)
    g, n = t.shape[-2:]
    return t if (n == 1 or t.stride(-1) == 1) and (g == 1 or t.stride(-2) == n) else _copy(t, name)


def _pair(B: torch.Tensor, C: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """In one type: in float32 where one is."""
    if B.dtype is not C.dtype:
        B, C = (t if t.dtype is torch.float32 else _copy(t, "B or C", dtype=torch.float32) for t in (B, C))
    return B, C


def _scan_desc(x, delta, A, B, C, D, gate, delta_bias, state, starts, lengths, softplus) -> StateSpaceDesc:
    batch, length, channels = x.shape
    x_batch, x_time, _ = x.stride()
    delta_batch, delta_time, _ = delta.stride()
    gate_batch, gate_time, _ = gate.stride() if gate is not None else (0, 0, 0)
    B_batch, B_time, _, _ = B.stride()
    C_batch, C_time, _, _ = C.stride()
    starts_batch, starts_time = starts.stride() if starts is not None else (0, 0)
    # (in the order of the fields)
    return StateSpaceDesc(
        x.data_ptr(), x_batch, x_time, delta.data_ptr(), delta_batch, delta_time, _p(gate), gate_batch, gate_time, A.data_ptr(),
        B.data_ptr(), B_batch, B_time, C.data_ptr(), C_batch, C_time, _p(D), _p(delta_bias), _p(state), _p(starts), starts_batch, starts_time,
        _p(lengths), None, 0, 0, None, None, batch, length, channels, A.shape[1], B.shape[2], _DTYPES[x.dtype], _DTYPES[B.dtype], softplus)


def _scan_scratch(desc: StateSpaceDesc, backward: int, device) -> torch.Tensor | None:
    need = c_int64()
    _abi.check(_scan_workspace(ctypes.byref(desc), backward, ctypes.byref(need)), "ilx_state_space_workspace")
    if need.value == 0:
        return None
    workspace = torch.empty(need.value, device=device)
    desc.workspace, desc.workspace_floats = workspace.data_ptr(), need.value
    return workspace


def _scan_call(x, delta, A, B, C, D, gate, delta_bias, state, starts, lengths, softplus, want_last, save=False):
    B, C = _pair(B, C)
    desc = _scan_desc(x, delta, A, B, C, D, gate, delta_bias, state, starts, lengths, softplus)
    batch, length, channels = x.shape
    device = x.device
    out = _empty_like(x)
    last = torch.empty(batch, A.shape[1], channels, device=device) if want_last else None
    saved = torch.empty(batch, (length + _BLOCK - 1) // _BLOCK, A.shape[1], channels, device=device) if save else None
    desc.out, desc.last, desc.saved = out.data_ptr(), _p(last), _p(saved)
    desc.out_batch, desc.out_time, _ = out.stride()
    workspace = _scan_scratch(desc, 0, device)
    _keep(x, delta, A, B, C, D, gate, delta_bias, state, starts, lengths, out, last, workspace)
    _launch(_scan_forward, desc, "ilx_state_space_forward", x.get_device())
    return out, last, saved, desc


class _StateSpaceScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, gate, delta_bias, state, starts, lengths, softplus, want_last):
        ctx.set_materialize_grads(False)
        out, last, saved, ctx.desc = _scan_call(x, delta, A, B, C, D, gate, delta_bias, state, starts, lengths, softplus, want_last, True)
        kept = (x, delta, A, B, C, D, gate, delta_bias, starts, lengths, saved)
        ctx.save_for_backward(*kept)
        ctx.places = _places(kept)
        ctx.has_state = state is not None
        return out, last

    @staticmethod
    @_once
    def backward(ctx, grad_out, grad_last):
        x, delta, A, B, C, D, gate, delta_bias, starts, lengths, saved = kept = ctx.saved_tensors
        d = ctx.desc
        rB, rC = _pair(B, C)
        if _places(kept) != ctx.places or rB is not B or rC is not C:   # (hooks may pack saved tensors and unpack them elsewhere)
            d = _scan_desc(x, delta, A, rB, rC, D, gate, delta_bias, None, starts, lengths, d.softplus)
            d.saved = saved.data_ptr()
        index, device = x.get_device(), x.device
        grad_out = torch.zeros_like(x) if grad_out is None else _check_activation(grad_out, "the output's gradient", x, index)
        grad_last = None if grad_last is None else grad_last.contiguous()
        gx, gA = _empty_like(x), torch.empty_like(A)
        gdelta, ggate = torch.empty_like(gx), None if gate is None else torch.empty_like(gx)
        gB, gC = torch.empty(rB.shape, dtype=rB.dtype, device=device), torch.empty(rC.shape, dtype=rC.dtype, device=device)
        gD, gbias = (None if t is None else torch.empty_like(t) for t in (D, delta_bias))
        gstate = torch.empty(x.shape[0], A.shape[1], x.shape[2], device=device) if ctx.has_state and ctx.needs_input_grad[8] else None
        d.grad_out, d.grad_x, d.grad_delta, d.grad_gate = grad_out.data_ptr(), gx.data_ptr(), gdelta.data_ptr(), _p(ggate)
        d.grad_out_batch, d.grad_out_time, _ = grad_out.stride()
        d.grad_batch, d.grad_time, _ = gx.stride()
        d.grad_last, d.grad_A, d.grad_B, d.grad_C = _p(grad_last), gA.data_ptr(), gB.data_ptr(), gC.data_ptr()
        d.grad_D, d.grad_delta_bias, d.grad_state = _p(gD), _p(gbias), _p(gstate)
        workspace = _scan_scratch(d, 1, device)  # noqa: F841  (alive until the launches are queued)
        _launch(_scan_backward, d, "ilx_state_space_backward", index)
        if rB is not B:
            gB = gB.to(B.dtype)
        if rC is not C:
            gC = gC.to(C.dtype)
        return gx, gdelta, gA, gB, gC, gD, ggate, gbias, gstate, None, None, None, None


def _scan_operands(x, index, delta, A, B, C, D, gate, delta_bias):
    channels = x.shape[-1]
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A has shape {tuple(A.shape)}, expected (channels, states) with 1..{MAX_STATES} states")
    states = A.shape[1]
    delta = _check_activation(delta, "delta", x, index)
    gate = None if gate is None else _check_activation(gate, "gate", x, index)
    A = _check_parameter(A, "A", (channels, states), index)
    D = _check_parameter(D, "D", (channels,), index)
    delta_bias = _check_parameter(delta_bias, "delta_bias", (channels,), index)
    B, C = _shared(B, "B", x, index), _shared(C, "C", x, index)
    groups, n = B.shape[-2:]
    if B.shape != C.shape or n != states or groups < 1 or channels % groups:
        raise ValueError(f"B {tuple(B.shape)} and C {tuple(C.shape)} must have {states} states and groups that divide {channels} channels")
    return delta, A, B, C, D, gate, delta_bias


def state_space_scan(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                     D: torch.Tensor | None = None, gate: torch.Tensor | None = None, delta_bias: torch.Tensor | None = None,
                     softplus: bool = True, state: torch.Tensor | None = None, starts: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None, return_state: bool = False):
    """Selective state space recurrence over time, per channel d (of group g) with N states::

        dt = softplus(delta + delta_bias)           (or the sum itself)
        h  = exp(dt * A[d]) * h + dt * B[b, t, g] * x,     y = (C[b, t, g] * h).sum() + D[d] * x
        out = y, or y * gate * sigmoid(gate)

    ``x``, ``delta``, ``gate`` (batch, length, channels); ``A`` (channels, N), N up to 32; ``B``, ``C`` (batch, length, groups, N)
    or (batch, length, N) shared by all channels, in x's type or float32; ``D``, ``delta_bias`` (channels).  ``state`` (batch,
    N, channels) is the state ahead of the first row (zeros if None); with ``return_state`` the result is ``(out, last)``.
    Differentiable in every operand but ``starts`` and ``lengths``; between a forward and its backward pass one state in 8
    rows is kept."""
    x, index = _check_x(x, 3)
    batch, length, channels = x.shape
    delta, A, B, C, D, gate, delta_bias = _scan_operands(x, index, delta, A, B, C, D, gate, delta_bias)
    state = _check_parameter(state, "state", (batch, A.shape[1], channels), index)
    starts = _check_starts(starts, (batch, length), index)
    lengths = _check_lengths(lengths, batch, length, index)
    args = (x, delta, A, B, C, D, gate, delta_bias, state, starts, lengths, 1 if softplus else 0, return_state)
    if _needs_gradients(args[:9]):
        out, last = _StateSpaceScan.apply(*args)
    else:
        out, last, _, _ = _scan_call(*args)
    return (out, last) if return_state else out


def state_space_step(x: torch.Tensor, delta: torch.Tensor, state: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                     D: torch.Tensor | None = None, gate: torch.Tensor | None = None, delta_bias: torch.Tensor | None = None,
                     softplus: bool = True, starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One row of :func:`state_space_scan` per sequence: ``x``, ``delta``, ``gate`` (batch, channels), ``B``, ``C`` (batch, groups,
    N) or (batch, N), ``state`` (batch, N, channels) updated in place, ``starts`` (batch) the environments whose episode begins
    with this row.  ``out`` may name the result's buffer, ``x``, ``delta`` or ``gate`` itself for one, and shares memory with no other operand."""
    x, index = _check_x(x, 2)
    _no_gradients("state_space_step", (x, delta, state, A, B, C, D, gate, delta_bias, out))
    batch, channels = x.shape
    delta, A, B, C, D, gate, delta_bias = _scan_operands(x, index, delta, A, B, C, D, gate, delta_bias)
    B, C = _pair(B, C)
    states = A.shape[1]
    _check_state(state, (batch, states, channels), index)
    starts = _check_starts(starts, (batch,), index)
    written = (state,) if out is None else (state, out)
    out = _check_out(out, x, state)
    _keep(x, delta, A, B, C, D, gate, delta_bias, state, starts, out)
    at = state.data_ptr()
    desc = StateSpaceDesc(
        x.data_ptr(), x.stride(0), 0, delta.data_ptr(), delta.stride(0), 0, _p(gate), gate.stride(0) if gate is not None else 0, 0, A.data_ptr(),
        B.data_ptr(), B.stride(0), 0, C.data_ptr(), C.stride(0), 0, _p(D), _p(delta_bias), at, _p(starts),
        starts.stride(0) if starts is not None else 0, 0, None, out.data_ptr(), out.stride(0), 0, at, None, batch, 1, channels, states, B.shape[1],
        _DTYPES[x.dtype], _DTYPES[B.dtype], 1 if softplus else 0)
    _launch(_scan_step, desc, "ilx_state_space_step", index)
    _written(written)
    return out
