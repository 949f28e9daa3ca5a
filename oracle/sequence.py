"""Oracle of the sequence operators: the definitions row by row in float64 on the CPU (differentiable by autograd), and the
magnitudes that bound the kernels' rounding: the same sums with every term's absolute value."""

from __future__ import annotations

import torch


def _gate(p):
    return p * torch.sigmoid(p)


def _softplus(v):
    return torch.logaddexp(v, torch.zeros_like(v))   # (a maximum and an absolute value would have slope 1 at exactly 0)


def _lengths(lengths, batch, length):
    return torch.full((batch,), length) if lengths is None else lengths.clamp(0, length)


def short_convolution(x, weight, bias=None, silu=False, state=None, starts=None, lengths=None):
    """(out, last); x (batch, length, channels), weight (channels, width)."""
    batch, length, channels = x.shape
    width = weight.shape[1]
    window = x.new_zeros(batch, width - 1, channels) if state is None else state
    end, outs = _lengths(lengths, batch, length), []
    for t in range(length):
        kept = window if starts is None else torch.where(starts[:, t, None, None].bool(), torch.zeros_like(window), window)
        rows = torch.cat([kept, x[:, t:t + 1]], 1)
        p = (rows * weight.t()).sum(1) + (0 if bias is None else bias)
        inside = t < end
        outs.append(torch.where(inside[:, None], _gate(p) if silu else p, torch.zeros_like(p)))
        window = torch.where(inside[:, None, None], rows[:, 1:], window)
    return (torch.stack(outs, 1) if outs else x), window


def state_space_scan(x, delta, A, B, C, D=None, gate=None, delta_bias=None, softplus=True, state=None, starts=None, lengths=None):
    """(out, last); B, C (batch, length, groups, states), state (batch, states, channels)."""
    batch, length, channels = x.shape
    groups, states = B.shape[2:]
    h = x.new_zeros(batch, states, channels) if state is None else state
    end, outs = _lengths(lengths, batch, length), []
    for t in range(length):
        raw = delta[:, t] + (0 if delta_bias is None else delta_bias)
        dt = _softplus(raw) if softplus else raw
        b, c = (v[:, t].repeat_interleave(channels // groups, 1).transpose(1, 2) for v in (B, C))
        kept = h if starts is None else torch.where(starts[:, t, None, None].bool(), torch.zeros_like(h), h)
        new = torch.exp(dt[:, None] * A.t()) * kept + (dt * x[:, t])[:, None] * b
        y = (c * new).sum(1) + (0 if D is None else D * x[:, t])
        if gate is not None:
            y = y * _gate(gate[:, t])
        inside = t < end
        outs.append(torch.where(inside[:, None], y, torch.zeros_like(y)))
        h = torch.where(inside[:, None, None], new, h)
    return (torch.stack(outs, 1) if outs else x), h


def _inside(x, lengths):
    return (torch.arange(x.shape[1])[None] < _lengths(lengths, x.shape[0], x.shape[1])[:, None])[..., None]


def short_convolution_magnitudes(x, weight, bias, silu, state, starts, lengths, grad_out, grad_last):
    """Per output the sum of the absolute values of its terms, an activation counted by its largest slope (1.1) and, in the
    gradients, by its own slope and what an error of p does to it (|act''| <= 1/2)."""
    leaves = dict(x=x.abs(), weight=weight.abs(), bias=torch.zeros(x.shape[2]).double() if bias is None else bias.abs(),
                  state=torch.zeros(x.shape[0], weight.shape[1] - 1, x.shape[2]).double() if state is None else state.abs())
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in leaves.items()}
    p, last = short_convolution(leaves["x"], leaves["weight"], leaves["bias"], False, leaves["state"], starts, lengths)
    out = 1.1 * p if silu else p
    through = grad_out.abs() * ((1.1 + 0.5 * p.detach()) if silu else 1.0)
    total = (p * through).sum() + (0 if grad_last is None else (last * grad_last.abs()).sum())
    grads = torch.autograd.grad(total, list(leaves.values()), allow_unused=True)
    found = {k: torch.zeros_like(v) if g is None else g for (k, v), g in zip(leaves.items(), grads)}
    return dict({"grad_" + k: g for k, g in found.items()}, out=out.detach(), last=last.detach())


def state_space_magnitudes(x, delta, A, B, C, D, gate, delta_bias, softplus, state, starts, lengths, grad_out, grad_last):
    """Per output the sum of the absolute values of its terms; decays keep their values."""
    batch, length, channels = x.shape
    groups, states = B.shape[2:]
    inside = _inside(x, lengths)
    raw = delta + (0 if delta_bias is None else delta_bias)
    dt = torch.where(inside, _softplus(raw) if softplus else raw, torch.zeros_like(raw))
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    xa = torch.where(inside, x, torch.zeros_like(x)).abs()
    a = torch.exp(dt[..., None] * A)                                           # (batch, length, channels, states)
    if starts is not None:
        a = torch.where((starts.bool() & inside[..., 0])[..., None, None], torch.zeros_like(a), a)
    Ba, Ca = (v.abs().repeat_interleave(channels // groups, 2) for v in (B, C))
    u = dt.abs() * xa
    h = torch.zeros(batch, channels, states).double() if state is None else state.abs().transpose(1, 2)
    p, hs = [], []
    for t in range(length):
        p.append(a[:, t] * h)
        h = p[-1] + u[:, t, :, None] * Ba[:, t]
        hs.append(h)
    found = dict(last=h.transpose(1, 2))
    if length == 0:
        return found
    p, hs = torch.stack(p, 1), torch.stack(hs, 1)
    Da = 0 if D is None else D.abs()
    y = (Ca * hs).sum(-1) + Da * xa
    go = torch.where(inside, grad_out, torch.zeros_like(grad_out)).abs()
    if gate is None:
        found["out"], dy = y, go
    else:
        sig = torch.sigmoid(gate)
        found["out"], dy = y * (gate * sig).abs(), go * (gate * sig).abs()
        found["grad_gate"] = go * y * sig * (1 + gate.abs() * (1 - sig))
    r, rs = (torch.zeros(batch, channels, states).double() if grad_last is None else grad_last.abs().transpose(1, 2)), [None] * length
    for t in reversed(range(length)):
        r = r + dy[:, t, :, None] * Ca[:, t]
        rs[t] = r
        r = r * a[:, t]
    rs = torch.stack(rs, 1)
    q, rb = rs * p, (rs * Ba).sum(-1)
    per_group = lambda v: v.reshape(batch, length, groups, channels // groups, states).sum(3)  # noqa: E731
    draw = torch.where(inside, (xa * rb + (q * A.abs()).sum(-1)) * slope, torch.zeros_like(raw))
    zero_rows = lambda v: torch.where(inside[..., None], v, torch.zeros_like(v))  # noqa: E731
    found.update(grad_x=torch.where(inside, Da * dy + dt.abs() * rb, torch.zeros_like(x)), grad_delta=draw, grad_A=(q * dt.abs()[..., None]).sum((0, 1)),
                 grad_B=zero_rows(per_group(rs * u[..., None])), grad_C=zero_rows(per_group(hs * dy[..., None])), grad_D=(dy * xa).sum((0, 1)),
                 grad_delta_bias=draw.sum((0, 1)), grad_state=r.transpose(1, 2))
    return found
