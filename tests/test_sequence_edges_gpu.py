"""GPU: calls of the sequence operators at the edges of what autograd, command lists and the argument types allow."""

import pytest
import torch
from torch.autograd import forward_ad

from isaaclab_amd import _abi
from isaaclab_amd.utils import sequence as S
from isaaclab_amd.utils.command_list import CommandList
from isaaclab_amd.utils.gradients import gradient_norm

pytestmark = pytest.mark.gpu


def operands(dev, batch=3, length=20, channels=24, states=4, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    return dict(x=r(batch, length, channels), delta=r(batch, length, channels), A=-torch.rand(channels, states, generator=gen).to(dev) - 0.5,
                B=r(batch, length, states), C=r(batch, length, states), D=r(channels), gate=r(batch, length, channels), delta_bias=r(channels),
                state=r(batch, states, channels))


def scan(v, **kw):
    return S.state_space_scan(v["x"], v["delta"], v["A"], v["B"], v["C"], D=v["D"], gate=v["gate"], delta_bias=v["delta_bias"], state=v["state"], **kw)


def step(v, t, state, **kw):
    return S.state_space_step(v["x"][:, t], v["delta"][:, t], state, v["A"], v["B"][:, t], v["C"][:, t], D=v["D"], gate=v["gate"][:, t],
                              delta_bias=v["delta_bias"], **kw)


def test_forward_mode_is_refused(dev):
    """Each operand in turn as a dual tensor: an error and not a result without its tangent."""
    v = operands(dev)
    conv = dict(x=v["x"], weight=torch.randn(24, 4, device=dev), bias=torch.randn(24, device=dev), state=torch.randn(3, 3, 24, device=dev))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for k in v:
            w = {**v, k: dual(v[k])}
            with pytest.raises(RuntimeError, match="forward-mode"):
                scan(w)
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():   # (which stops reverse mode only)
                step(w, 0, w["state"])
        for k in conv:
            w = {**conv, k: dual(conv[k])}
            with pytest.raises(RuntimeError, match="forward-mode"):
                S.short_convolution(w["x"], w["weight"], w["bias"], state=w["state"])
            with pytest.raises(RuntimeError, match="forward-mode"):
                S.short_convolution_step(w["x"][:, 0], w["state"], w["weight"], w["bias"])
        inside = scan(v)
    assert torch.equal(inside, scan(v))


def test_out_is_written_in_sight_of_autograd(dev):
    """A buffer that a graph has saved and a step then writes fails the backward pass; a leaf that needs gradients is refused."""
    v, weight = operands(dev), torch.randn(24, 4, device=dev)
    conv = torch.zeros(3, 3, 24, device=dev)
    for call in (lambda out: S.short_convolution_step(v["x"][:, 0], conv, weight, out=out), lambda out: step(v, 0, v["state"], out=out)):
        for buffer in (torch.ones(5, 3, 24, device=dev)[2], torch.ones(3, 30, device=dev)[:, :24]):
            leaf = torch.ones(3, 24, device=dev, requires_grad=True)
            product = (leaf * buffer).sum()
            before = buffer._version
            with torch.no_grad():
                assert call(buffer) is buffer
            assert buffer._version > before
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                torch.autograd.grad(product, leaf)
        leaf = torch.ones(3, 24, device=dev, requires_grad=True)
        with pytest.raises(RuntimeError, match="no backward"):
            call(leaf)
        assert torch.equal(leaf, torch.ones_like(leaf))
        with torch.inference_mode():
            call(torch.empty(3, 24, device=dev))


def test_out_in_the_place_of_an_operand(dev):
    """x, delta or gate may be the result's buffer; the state may not, not even in part."""
    for channels in (24, 130, 61):
        v, weight = operands(dev, batch=9000, length=1, channels=channels), torch.randn(channels, 4, device=dev)
        rows = lambda k: v[k][:, 0].clone()  # noqa: E731
        for name in ("x", "delta", "gate"):
            w = {k: rows(k) for k in ("x", "delta", "gate", "B", "C")}
            s1, s2 = v["state"].clone(), v["state"].clone()
            args = lambda s: (w["x"], w["delta"], s, v["A"], w["B"], w["C"])  # noqa: E731
            want = S.state_space_step(*args(s1), D=v["D"], gate=w["gate"], delta_bias=v["delta_bias"])
            got = S.state_space_step(*args(s2), D=v["D"], gate=w["gate"], delta_bias=v["delta_bias"], out=w[name])
            assert got is w[name] and torch.equal(got, want) and torch.equal(s1, s2)
        s1, s2, x = torch.randn(9000, 3, channels, device=dev), None, rows("x")
        s2 = s1.clone()
        want = S.short_convolution_step(x, s1, weight, activation="silu")
        assert torch.equal(S.short_convolution_step(x, s2, weight, activation="silu", out=x), want) and torch.equal(s1, s2)
    block = torch.zeros(3 * 4 * 24 + 40, device=dev)
    state, over = block[:3 * 4 * 24].view(3, 4, 24), block[-3 * 24:].view(3, 24)
    v = operands(dev)
    with pytest.raises(ValueError, match="share memory"):
        step(v, 0, state, out=over)
    state = block[:3 * 3 * 24].view(3, 3, 24)
    with pytest.raises(ValueError, match="share memory"):
        S.short_convolution_step(v["x"][:, 0], state, torch.randn(24, 4, device=dev), out=state[:, 1])
    assert not block.any()


def test_lengths_past_32_bits(dev):
    """64-bit lengths are clamped as they are, not as what is left of them in 32 bits."""
    v, weight = operands(dev), torch.randn(24, 4, device=dev)
    lengths = torch.tensor([2 ** 32 + 5, torch.iinfo(torch.int64).max, -2 ** 40 + 7], device=dev)
    clamped = torch.tensor([20, 20, 0], dtype=torch.int32, device=dev)
    for call in (lambda n: scan(v, lengths=n, return_state=True), lambda n: S.short_convolution(v["x"], weight, lengths=n, return_state=True)):
        assert all(torch.equal(a, b) for a, b in zip(call(lengths), call(clamped)))
    assert torch.equal(scan(v, lengths=lengths)[:2], scan(v)[:2])


def test_a_command_list_holds_what_its_calls_read(dev):
    """Operands that only the recorded call named: their memory stays theirs until the list goes."""
    v, weight = operands(dev), torch.randn(24, 4, device=dev)
    flags, lengths = torch.zeros(3, 20, device=dev), torch.tensor([3, 20, 11], dtype=torch.int32, device=dev)
    flags[:, 9] = 1.0
    conv, state = torch.zeros(3, 3, 24, device=dev), v["state"].clone()
    copies = lambda: {k: t.clone() for k, t in v.items()}  # noqa: E731

    def calls(conv, state):
        yield scan(copies(), starts=flags > 0, lengths=lengths + 0, return_state=True)
        yield S.short_convolution(v["x"] + 0, weight + 0, state=conv + 1, starts=flags > 0, lengths=lengths + 0, return_state=True)
        yield (S.short_convolution_step(v["x"][:, 0] + 0, conv, weight + 0, starts=flags[:, 9] > 0),)
        yield (step(copies(), 0, state, starts=flags[:, 9] > 0),)
        yield (gradient_norm([v["x"] + 0, weight + 0]),)

    commands = CommandList()
    with torch.no_grad(), commands.record():
        recorded = [call for call in calls(conv, state)]
        junk = [torch.full((n,), float("nan"), device=dev) for n in (12, 24, 72, 96, 240, 288, 1440) for _ in range(40)]
    commands.replay()
    fresh_conv, fresh_state = torch.zeros_like(conv), v["state"].clone()
    for got, want in zip(recorded, calls(fresh_conv, fresh_state)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(conv, fresh_conv) and torch.equal(state, fresh_state)
    del junk


def test_a_backward_pass_is_not_recorded(dev):
    """Autograd on the recording thread itself: refused, where the launches would be kept and the gradients left unwritten."""
    v, weight = operands(dev), torch.randn(24, 4, device=dev)
    for call in (lambda x: S.short_convolution(x, weight), lambda x: scan({**v, "x": x})):
        x = v["x"].clone().requires_grad_(True)
        out = call(x)
        with torch.autograd.set_multithreading_enabled(False):
            with CommandList().record(), pytest.raises(_abi.IlxError, match="backward pass cannot be recorded"):
                torch.autograd.grad(out.sum(), x, retain_graph=True)
            same_thread, = torch.autograd.grad(out.sum(), x, retain_graph=True)
        assert torch.equal(same_thread, torch.autograd.grad(out.sum(), x)[0])


@pytest.mark.parametrize("lo,hi", [(-85.0, -40.0), (-40.0, -20.0), (-20.0, -10.0), (-10.0, -3.0), (-3.0, -1.0), (-1.0, 0.0), (0.0, 1.0), (1.0, 30.0)])
def test_softplus_relative_error(dev, lo, hi):
    """The step size keeps its relative accuracy however small it is: dt = softplus(delta) itself, by x = B = C = 1 and no state.
    In units of 2^-24: 9 + 1.3 |delta| below zero (the exponent's rounding), 9 above."""
    rows, channels = 64, 1024
    delta = torch.rand(1, rows, channels, generator=torch.Generator().manual_seed(int(lo))).to(dev) * (hi - lo) + lo
    starts = torch.ones(1, rows, dtype=torch.bool, device=dev)
    one = torch.ones(1, rows, 1, device=dev)
    dt = S.state_space_scan(torch.ones_like(delta), delta, torch.zeros(channels, 1, device=dev), one, one, starts=starts)
    x = delta.double()
    want = x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))
    units = (dt.double() / want - 1).abs() * 2 ** 24
    bound = 9 + 1.3 * (-x).clamp(min=0)
    print(f"softplus on [{lo}, {hi}]: {float(units.max()):.1f} units")
    assert (units <= bound).all(), float((units / bound).max())
