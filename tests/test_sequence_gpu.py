"""GPU: the sequence operators (short causal convolution, selective state space recurrence) against the float64 oracle.

Tolerances.  The kernels compute in float32, so an output is off by at most n u M: u = 2^-24, M the sum of the absolute values
of the terms it is made of (the oracle's magnitudes) and n the roundings on the longest path to it.  Convolution: W + 1
products and a gate of at most 40 roundings; a parameter's gradient adds a rounding for each row it sums.  Recurrence:
softplus, product and gate are at most 60 roundings; a row's decay exp(dt A) is off by (40 |dt A| + 2) u, of which
|dt A| exp(-|dt A|) <= 0.37 reaches the state, so at most 20 u per row, and the same again on the way back.  A 16-bit result is
rounded once more, by at most half a step of its type.  Sums over channels, states and rows add a rounding for each term.
"""

import pytest
import torch
import torch.utils.checkpoint

from isaaclab_amd import _abi
from isaaclab_amd.utils import sequence as S
from isaaclab_amd.utils.command_list import CommandList
from oracle import sequence as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(got, ref, magnitude, n, what):
    """|got - ref| <= n u M, and half a step of a 16-bit result."""
    got = got.detach().cpu()
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} != {tuple(ref.shape)}"
    bound = n * U * magnitude + 1e-37
    if got.dtype != torch.float32:
        bound = bound + torch.finfo(got.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    off = (got.double() - ref).abs()
    bad = ~(off <= bound)
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {float(got[at])} for {float(ref[at])}, bound {float(bound[at]):.3g}")


def rows(gen, batch, length, tail, dtype, time_major, scale=1.0):
    """(batch, length, tail) values in ``dtype``, as a recorder's time-major buffer where asked."""
    lead = (length, batch) if time_major else (batch, length)
    t = (torch.randn(*lead, *tail, generator=gen) * scale).to(dtype)
    return t.transpose(0, 1) if time_major else t


def leaves_of(dev, **tensors):
    """GPU copies (with their strides) that need gradients, and float64 copies for the oracle."""
    gpu = {k: None if t is None else t.to(dev).requires_grad_(True) for k, t in tensors.items()}
    ref = {k: None if t is None else t.detach().double().requires_grad_(True) for k, t in tensors.items()}
    return gpu, ref


def flags_of(gen, batch, length, with_starts, with_lengths, time_major):
    starts = lengths = None
    if with_starts:
        starts = rows(gen, batch, length, (), torch.float32, time_major) > 1.0
    if with_lengths:
        lengths = torch.randint(0, length + 1, (batch,), generator=gen, dtype=torch.int32)
    return starts, lengths


# ---- convolution ----------------------------------------------------------------------------------------------------
CONV = [  # batch, length, channels, width, dtype, silu, starts, lengths, state, time major
    (1, 1, 1, 1, 0, False, False, False, False, False),
    (2, 3, 5, 2, 0, True, False, False, True, False),
    (1, 2, 8, 8, 0, True, True, False, True, False),
    (3, 33, 20, 4, 0, True, True, True, True, False),
    (2, 70, 64, 4, 0, False, True, False, False, True),
    (4, 24, 256, 4, 0, True, True, False, True, True),
    (1, 129, 100, 8, 1, True, False, True, True, False),
    (5, 31, 12, 3, 1, True, True, False, True, True),
    (2, 65, 36, 5, 2, True, True, True, False, False),
    (2, 32, 300, 7, 2, False, False, False, True, False),
    (3, 64, 7, 6, 1, True, True, True, True, True),
    (2, 300, 520, 4, 1, True, True, True, True, False),
    # enough rows for four or eight channels a thread, whole and overlapping at the end of a row
    (300, 8, 1801, 4, 0, True, True, True, True, True),
    (600, 5, 1803, 3, 1, True, True, True, True, False),
    (550, 6, 2048, 4, 1, True, True, False, True, True),
    (1100, 16, 258, 8, 2, True, False, True, False, False),
    (24, 180, 1210, 4, 1, True, True, True, True, False),
    (300, 8, 1800, 2, 0, False, False, False, True, False),
]


@pytest.mark.parametrize("batch,length,channels,width,dtype,silu,with_starts,with_lengths,with_state,time_major", CONV)
def test_convolution_and_its_gradients(dev, batch, length, channels, width, dtype, silu, with_starts, with_lengths, with_state, time_major):
    gen = torch.Generator().manual_seed(length * 31 + channels)
    dt = DTYPES[dtype]
    starts, lengths = flags_of(gen, batch, length, with_starts, with_lengths, time_major)
    gpu, ref = leaves_of(dev, x=rows(gen, batch, length, (channels,), dt, time_major), weight=torch.randn(channels, width, generator=gen) * 0.5,
                         bias=torch.randn(channels, generator=gen), state=torch.randn(batch, width - 1, channels, generator=gen) if with_state else None)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    out, last = S.short_convolution(gpu["x"], gpu["weight"], gpu["bias"], activation="silu" if silu else None, state=gpu["state"], starts=on(starts),
                                    lengths=on(lengths), return_state=True)
    ref_out, ref_last = O.short_convolution(ref["x"], ref["weight"], ref["bias"], silu, ref["state"], starts, lengths)
    g, gl = rows(gen, batch, length, (channels,), dt, False), torch.randn(batch, width - 1, channels, generator=gen)
    names = [k for k in gpu if gpu[k] is not None]
    m = O.short_convolution_magnitudes(ref["x"].detach(), ref["weight"].detach(), ref["bias"].detach(), silu,
                                       None if ref["state"] is None else ref["state"].detach(), starts, lengths, g.double(), gl.double())
    assert out.dtype == dt and out.stride() == torch.empty_like(gpu["x"]).stride()
    close(out, ref_out.detach(), m["out"], 40 + width, "out")
    assert torch.equal(last.detach().cpu().double(), ref_last.detach()), "the carried state holds inputs as they are"
    got = torch.autograd.grad([out, last], [gpu[k] for k in names], [g.to(dev), gl.to(dev)], allow_unused=width == 1)
    want = torch.autograd.grad([ref_out, ref_last], [ref[k] for k in names], [g.double(), gl.double()], allow_unused=True)
    for k, a, b in zip(names, got, want):
        if b is None:
            continue
        close(a, b, m["grad_" + k], 80 + 2 * width + (batch * length if k in ("weight", "bias") else 0), f"gradient of {k}")
    plain = S.short_convolution(gpu["x"].detach(), gpu["weight"].detach(), gpu["bias"].detach(), activation="silu" if silu else None,
                                state=on(None if gpu["state"] is None else gpu["state"].detach()), starts=on(starts), lengths=on(lengths))
    assert torch.equal(plain, out.detach()) and not plain.requires_grad


def test_convolution_steps_are_the_sequence(dev):
    """Any cut of a sequence, down to single rows, gives the same bits."""
    gen = torch.Generator().manual_seed(5)
    for dt in DTYPES:
        x = torch.randn(6, 19, 44, generator=gen).to(dev, dt)
        w, b, s = (torch.randn(*shape, generator=gen).to(dev) for shape in ((44, 4), (44,), (6, 3, 44)))
        starts = (torch.rand(6, 19, generator=gen) < 0.2).to(dev)
        out, last = S.short_convolution(x, w, b, activation="silu", state=s, starts=starts, return_state=True)
        o1, mid = S.short_convolution(x[:, :7], w, b, activation="silu", state=s, starts=starts[:, :7], return_state=True)
        o2, end = S.short_convolution(x[:, 7:], w, b, activation="silu", state=mid, starts=starts[:, 7:], return_state=True)
        assert torch.equal(torch.cat([o1, o2], 1), out) and torch.equal(end, last)
        state = s.clone()
        for t in range(19):
            o = S.short_convolution_step(x[:, t], state, w, b, activation="silu", starts=starts[:, t])
            assert torch.equal(o, out[:, t]), (dt, t)
        assert torch.equal(state, last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,channels,width", [(1, 1, 1), (1, 256, 4), (7, 30, 2), (1000, 36, 4), (3, 1025, 8), (5, 12, 5), (9000, 61, 4), (20000, 61, 3), (20000, 64, 2), (17000, 30, 8)])
def test_convolution_step(dev, dtype, batch, channels, width):
    gen = torch.Generator().manual_seed(batch + channels)
    x, w = torch.randn(batch, channels, generator=gen).to(dtype), torch.randn(channels, width, generator=gen)
    s, starts = torch.randn(batch, width - 1, channels, generator=gen), torch.rand(batch, generator=gen) < 0.3
    state, out = s.to(dev), torch.empty(batch, channels + 3, dtype=dtype, device=dev)[:, :channels]
    got = S.short_convolution_step(x.to(dev), state, w.to(dev), activation="silu", starts=starts.to(dev), out=out)
    assert got is out
    ref, last = O.short_convolution(x.double()[:, None], w.double(), None, True, s.double(), starts[:, None])
    m = O.short_convolution_magnitudes(x.double()[:, None], w.double(), None, True, s.double(), starts[:, None], None, torch.ones(batch, 1, channels).double(), None)
    close(out, ref[:, 0], m["out"][:, 0], 40 + width, "out")
    assert torch.equal(state.cpu().double(), last)


# ---- recurrence -----------------------------------------------------------------------------------------------------
SCAN = [  # batch, length, channels, states, groups, dtype, shared in float32, gate, softplus, starts, lengths, state, time major
    (1, 1, 1, 1, 1, 0, False, False, True, False, False, False, False),
    (2, 5, 3, 2, 1, 0, False, True, True, True, False, True, False),
    (3, 37, 20, 5, 1, 0, False, False, True, True, True, True, True),
    (2, 16, 64, 16, 1, 0, False, True, True, False, False, True, False),
    (2, 17, 130, 16, 2, 0, False, True, True, True, False, False, True),
    (1, 64, 65, 8, 1, 1, False, True, True, False, True, True, False),
    (5, 24, 96, 11, 3, 1, False, True, True, True, False, True, True),
    (2, 33, 48, 32, 1, 1, True, True, True, True, True, True, False),
    (3, 40, 40, 20, 2, 2, False, False, True, True, False, True, False),
    (1, 100, 64, 4, 1, 2, False, True, False, False, True, False, True),
    (40, 24, 64, 16, 1, 0, False, True, True, True, False, True, True),
    (2, 130, 72, 16, 1, 0, False, False, False, True, True, True, False),
    (1, 700, 32, 16, 1, 0, False, True, True, False, False, True, False),
    (3, 555, 24, 6, 1, 1, False, True, True, True, True, True, False),
    (2, 333, 70, 24, 2, 1, True, True, True, True, True, True, True),
    (1, 520, 40, 32, 1, 0, False, True, False, False, False, True, False),
    (2, 96, 12, 3, 4, 2, False, False, True, True, False, False, False),
]


def scan_inputs(gen, batch, length, channels, states, groups, dt, shared_f32, with_gate, softplus, with_state, time_major):
    shared = torch.float32 if shared_f32 else dt
    tensors = dict(
        x=rows(gen, batch, length, (channels,), dt, time_major), delta=rows(gen, batch, length, (channels,), dt, time_major, 0.7),
        A=-torch.exp(torch.rand(channels, states, generator=gen) * 3 - 1), B=rows(gen, batch, length, (groups, states), shared, time_major),
        C=rows(gen, batch, length, (groups, states), shared, time_major), D=torch.randn(channels, generator=gen),
        gate=rows(gen, batch, length, (channels,), dt, time_major) if with_gate else None, delta_bias=torch.randn(channels, generator=gen) - 2,
        state=torch.randn(batch, states, channels, generator=gen) if with_state else None)
    if not softplus:   # the step itself: positive
        tensors["delta"] = tensors["delta"].abs() * 0.3
        tensors["delta_bias"] = tensors["delta_bias"].abs() * 0.01
    return tensors


ORDER = ("x", "delta", "A", "B", "C", "D", "gate", "delta_bias", "softplus", "state", "starts", "lengths")


def oracle_args(ref, softplus, starts, lengths, detach=False):
    known = dict(ref, softplus=softplus, starts=starts, lengths=lengths)
    return [known[k].detach() if detach and isinstance(known[k], torch.Tensor) else known[k] for k in ORDER]


@pytest.mark.parametrize("batch,length,channels,states,groups,dtype,shared_f32,with_gate,softplus,with_starts,with_lengths,with_state,time_major", SCAN)
def test_scan_and_its_gradients(dev, batch, length, channels, states, groups, dtype, shared_f32, with_gate, softplus, with_starts, with_lengths,
                                with_state, time_major):
    gen = torch.Generator().manual_seed(length * 17 + channels)
    dt = DTYPES[dtype]
    starts, lengths = flags_of(gen, batch, length, with_starts, with_lengths, time_major)
    gpu, ref = leaves_of(dev, **scan_inputs(gen, batch, length, channels, states, groups, dt, shared_f32, with_gate, softplus, with_state, time_major))
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    call = lambda v, **kw: S.state_space_scan(v["x"], v["delta"], v["A"], v["B"], v["C"], D=v["D"], gate=v["gate"], delta_bias=v["delta_bias"],  # noqa: E731
                                              softplus=softplus, state=v["state"], starts=on(starts), lengths=on(lengths), **kw)
    out, last = call(gpu, return_state=True)
    ref_out, ref_last = O.state_space_scan(*oracle_args(ref, softplus, starts, lengths))
    g, gl = rows(gen, batch, length, (channels,), dt, time_major), torch.randn(batch, states, channels, generator=gen)
    m = O.state_space_magnitudes(*oracle_args(ref, softplus, starts, lengths, True), g.double(), gl.double())
    n = 60 + 20 * length + states
    close(last, ref_last.detach(), m["last"], n, "last")
    close(out, ref_out.detach(), m["out"], n, "out")
    names = [k for k in gpu if gpu[k] is not None]
    got = torch.autograd.grad([out, last], [gpu[k] for k in names], [g.to(dev), gl.to(dev)])
    want = torch.autograd.grad([ref_out, ref_last], [ref[k] for k in names], [g.double(), gl.double()])
    for k, a, b in zip(names, got, want):
        terms = {"A": batch * length, "D": batch * length, "delta_bias": batch * length, "B": channels, "C": channels}.get(k, 0)
        assert a.dtype == gpu[k].dtype
        close(a, b, m["grad_" + k], 2 * n + terms, f"gradient of {k}")
    detached = {k: None if v is None else v.detach() for k, v in gpu.items()}
    plain = call(detached)
    close(plain, ref_out.detach(), m["out"], n, "out without gradients")
    assert not plain.requires_grad
    again = call(gpu, return_state=True)
    twice = torch.autograd.grad(again, [gpu[k] for k in names], [g.to(dev), gl.to(dev)])
    assert all(torch.equal(a, b) for a, b in zip(got, twice)), "two runs give the same bits"


def test_scan_steps_are_the_sequence(dev):
    """Single rows follow the sequence (same arithmetic per row, so the same bound), and so does a cut in two."""
    gen = torch.Generator().manual_seed(8)
    for dt in DTYPES:
        v = scan_inputs(gen, 5, 21, 70, 16, 1, dt, False, True, True, True, False)
        starts = torch.rand(5, 21, generator=gen) < 0.15
        ref = {k: t.double() for k, t in v.items()}
        ref_out, ref_last = O.state_space_scan(*oracle_args(ref, True, starts, None))
        m = O.state_space_magnitudes(*oracle_args(ref, True, starts, None), torch.zeros(5, 21, 70).double(), None)
        n = 60 + 20 * 21 + 16
        v, starts = {k: t.to(dev) for k, t in v.items()}, starts.to(dev)
        kw = dict(D=v["D"], delta_bias=v["delta_bias"])
        state = v["state"].clone()
        for t in range(21):
            o = S.state_space_step(v["x"][:, t], v["delta"][:, t], state, v["A"], v["B"][:, t], v["C"][:, t], gate=v["gate"][:, t], starts=starts[:, t], **kw)
            close(o, ref_out[:, t], m["out"][:, t], n, f"step {t}")
        close(state, ref_last, m["last"], n, "state")
        part = lambda a, b: [v[k][:, a:b] for k in ("x", "delta")] + [v["A"]] + [v[k][:, a:b] for k in ("B", "C")]  # noqa: E731
        o1, mid = S.state_space_scan(*part(0, 9), gate=v["gate"][:, :9], state=v["state"], starts=starts[:, :9], return_state=True, **kw)
        o2, end = S.state_space_scan(*part(9, 21), gate=v["gate"][:, 9:], state=mid, starts=starts[:, 9:], return_state=True, **kw)
        close(torch.cat([o1, o2], 1), ref_out, m["out"], n, "cut in two")
        close(end, ref_last, m["last"], n, "state of the second part")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,channels,states,groups", [(1, 1, 1, 1), (1, 256, 16, 1), (9, 130, 16, 2), (700, 40, 5, 1), (4, 100, 32, 1), (33, 96, 12, 3), (5000, 64, 16, 1)])
def test_scan_step(dev, dtype, batch, channels, states, groups):
    gen = torch.Generator().manual_seed(batch + channels)
    v = scan_inputs(gen, batch, 1, channels, states, groups, dtype, False, True, True, True, False)
    starts = torch.rand(batch, 1, generator=gen) < 0.3
    ref = {k: t.double() for k, t in v.items()}
    ref_out, ref_last = O.state_space_scan(*oracle_args(ref, True, starts, None))
    m = O.state_space_magnitudes(*oracle_args(ref, True, starts, None), torch.zeros(batch, 1, channels).double(), None)
    v = {k: t.to(dev) for k, t in v.items()}
    state = v["state"].clone()
    out = S.state_space_step(v["x"][:, 0], v["delta"][:, 0], state, v["A"], v["B"][:, 0], v["C"][:, 0], D=v["D"], gate=v["gate"][:, 0],
                             delta_bias=v["delta_bias"], starts=starts[:, 0].to(dev))
    close(out, ref_out[:, 0], m["out"][:, 0], 80 + states, "out")
    close(state, ref_last, m["last"], 80 + states, "state")


# ---- where it can go wrong --------------------------------------------------------------------------------------------
def some(dev, batch=3, length=40, channels=68, states=16, dt=torch.float32, seed=3):
    gen = torch.Generator().manual_seed(seed)
    v = scan_inputs(gen, batch, length, channels, states, 1, dt, False, True, True, True, False)
    return {k: t.to(dev) for k, t in v.items()}


def run_scan(v, **kw):
    return S.state_space_scan(v["x"], v["delta"], v["A"], v["B"], v["C"], D=v["D"], gate=v["gate"], delta_bias=v["delta_bias"], state=v["state"],
                              return_state=True, **kw)


def test_rows_behind_the_end_are_not_read(dev):
    v = some(dev)
    lengths = torch.tensor([0, 17, 40], device=dev)
    clean = run_scan(v, lengths=lengths)
    dirty = {k: t.clone() for k, t in v.items()}
    for b, n in enumerate(lengths.tolist()):
        for k in ("x", "delta", "gate", "B", "C"):
            dirty[k][b, n:] = float("nan")
    leaves = {k: t.requires_grad_(True) for k, t in dirty.items()}
    out, last = run_scan(leaves, lengths=lengths)
    assert torch.equal(out, clean[0]) and torch.equal(last, clean[1])
    assert torch.equal(last[0], v["state"][0]) and not out[0].any() and not out[1, 17:].any()
    grads = torch.autograd.grad([out, last], list(leaves.values()), [torch.ones_like(out), torch.ones_like(last)])
    for k, g in zip(leaves, grads):
        assert torch.isfinite(g).all(), k
        if k in ("x", "delta", "gate", "B", "C"):
            assert not g[0].any() and not g[1, 17:].any(), k
    assert torch.equal(grads[list(leaves).index("state")][0], torch.ones_like(last[0]))
    # and the convolution
    w = torch.randn(68, 4, device=dev)
    s = torch.randn(3, 3, 68, device=dev)
    clean = S.short_convolution(v["x"].detach(), w, state=s, lengths=lengths, return_state=True)
    x, w, s = dirty["x"].detach().requires_grad_(True), w.requires_grad_(True), s.requires_grad_(True)
    out, last = S.short_convolution(x, w, state=s, lengths=lengths, return_state=True)
    assert torch.equal(out, clean[0]) and torch.equal(last, clean[1]) and torch.equal(last[0], s[0])
    gx, gw, gs = torch.autograd.grad([out, last], [x, w, s], [torch.ones_like(out), torch.ones_like(last)])
    assert torch.isfinite(gw).all() and not gx[0].any() and not gx[1, 17:].any() and torch.equal(gs[0], torch.ones_like(gs[0]))


def test_a_start_hides_what_was_before_it(dev):
    """Infinities and NaN in the carried state and in earlier rows do not pass a start; a start on every row is no memory."""
    v = some(dev)
    starts = torch.zeros(3, 40, dtype=torch.bool, device=dev)
    starts[:, 11] = True
    clean = run_scan(v, starts=starts)
    bad = {k: t.clone() for k, t in v.items()}
    bad["state"].fill_(float("nan"))
    bad["x"][:, :11] = float("inf")
    out, last = run_scan(bad, starts=starts)
    assert torch.equal(out[:, 11:], clean[0][:, 11:]) and torch.equal(last, clean[1])
    w, s = torch.randn(68, 4, device=dev), torch.full((3, 3, 68), float("nan"), device=dev)
    out, last = S.short_convolution(bad["x"], w, state=s, starts=starts, return_state=True)
    clean = S.short_convolution(v["x"], w, starts=starts, return_state=True)
    assert torch.equal(out[:, 11:], clean[0][:, 11:]) and torch.equal(last, clean[1])
    step = s.clone()
    S.short_convolution_step(v["x"][:, 0], step, w, starts=torch.ones(3, dtype=torch.uint8, device=dev))
    assert torch.equal(step, torch.cat([torch.zeros(3, 2, 68, device=dev), v["x"][:, :1]], 1))
    every = torch.ones_like(starts)
    out, last = S.short_convolution(v["x"], w, starts=every, return_state=True)
    assert torch.equal(out, v["x"] * w[:, 3]) and not last[:, :2].any()
    bad = {k: t.clone() for k, t in v.items()}
    bad["state"].fill_(float("nan"))
    assert torch.equal(run_scan(bad, starts=every)[0], run_scan(dict(v, state=torch.zeros_like(v["state"])), starts=every)[0])


def test_lengths_are_clamped_and_empty_shapes_pass(dev):
    v = some(dev)
    full = run_scan(v)
    over = run_scan(v, lengths=torch.tensor([40, 1000, 41], device=dev))
    assert torch.equal(over[0], full[0]) and torch.equal(over[1], full[1])
    none = run_scan(v, lengths=torch.tensor([-5, 0, -1], device=dev))
    assert not none[0].any() and torch.equal(none[1], v["state"])
    for batch, length in ((0, 5), (2, 0)):
        x = torch.zeros(batch, length, 8, device=dev, requires_grad=True)
        w = torch.ones(8, 4, device=dev, requires_grad=True)
        s = torch.ones(batch, 3, 8, device=dev, requires_grad=True)
        out, last = S.short_convolution(x, w, state=s, return_state=True)
        assert out.shape == x.shape and torch.equal(last, s)
        gw, gs = torch.autograd.grad(last.sum() + out.sum(), [w, s])
        assert not gw.any() and torch.equal(gs, torch.ones_like(s))
        b = torch.zeros(batch, length, 4, device=dev)
        h = torch.ones(batch, 4, 8, device=dev, requires_grad=True)
        out, last = S.state_space_scan(x, x, -w, b, b, state=h, return_state=True)
        assert out.shape == x.shape and torch.equal(last, h)
        ga, gh = torch.autograd.grad(last.sum() + out.sum(), [w, h])
        assert not ga.any() and torch.equal(gh, torch.ones_like(h))


def test_strides_and_alignment(dev):
    """Column ranges of wider rows, odd addresses, expanded batches and permuted layouts give what dense copies give."""
    gen = torch.Generator().manual_seed(4)
    for dt in DTYPES:
        wide = torch.randn(4, 20, 203, generator=gen).to(dev, dt)
        w, b = torch.randn(64, 4, generator=gen).to(dev), torch.randn(64, generator=gen).to(dev)
        for x in (wide[..., 3:67], wide[..., 4:68], wide[:1, :, 5:69].expand(4, 20, 64), wide.transpose(0, 1)[..., 1:65].transpose(0, 1),
                  wide[:, ::2, 64:128], wide[..., :128:2]):
            dense = x.contiguous()
            assert torch.equal(S.short_convolution(x, w, b, activation="silu"), S.short_convolution(dense, w, b, activation="silu"))
            x1, x2 = x.detach().requires_grad_(True), dense.detach().clone().requires_grad_(True)
            g1, = torch.autograd.grad(S.short_convolution(x1, w, b, activation="silu").float().sum(), x1)
            g2, = torch.autograd.grad(S.short_convolution(x2, w, b, activation="silu").float().sum(), x2)
            assert torch.equal(g1, g2)
        v = some(dev, batch=4, length=20, channels=64, dt=dt)
        bc = torch.randn(4, 20, 70, generator=gen).to(dev, dt)
        for off in (0, 1, 2, 37):
            B, C = bc[..., off:off + 16], bc[..., off + 16:off + 32]
            kw = dict(D=v["D"], delta_bias=v["delta_bias"])
            ref = S.state_space_scan(v["x"], v["delta"], v["A"], B.contiguous(), C.contiguous(), gate=v["gate"], **kw)
            got = S.state_space_scan(wide_of(v["x"]), wide_of(v["delta"]), v["A"], B, C, gate=wide_of(v["gate"]), **kw)
            assert torch.equal(ref, got), (dt, off)


def test_sliding_windows_over_one_series(dev):
    """x as overlapping rows of one series: time and channels both have stride 1, and so may the batch."""
    series = torch.randn(3, 60, device=dev)
    weight = torch.randn(20, 3, device=dev)
    for view in (series.unfold(1, 20, 1), series[0].unfold(0, 20, 1).unfold(0, 4, 1).transpose(1, 2)):
        assert view.stride(1) == 1 and view.stride(2) == 1
        batch, length, _ = view.shape
        v = some(dev, batch=batch, length=length, channels=20, states=4)
        results = []
        for x in (view, view.contiguous()):
            x = x.detach().requires_grad_(True)
            state = torch.zeros(batch, 2, 20, device=dev)
            out = S.short_convolution(x, weight, activation="silu")
            y, _ = run_scan({**v, "x": x})
            with torch.no_grad():
                step = S.short_convolution_step(x[:, 0], state, weight)
            results.append((out, y, *torch.autograd.grad(out.square().sum() + y.square().sum(), x), step, state))
        for got, plain in zip(*results):
            assert torch.equal(got, plain)


@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_rows_of_many_channels(dev, dtype):
    """Slices that begin at any element and rows of odd lengths, at sizes that take several channels a thread."""
    wide = torch.randn(800, 8, 1611, device=dev).to(dtype)
    weight, bias = torch.randn(1600, 4, device=dev, requires_grad=True), torch.randn(1600, device=dev)
    grad = torch.randn(800, 8, 1605, device=dev).to(dtype)
    results = []
    for x, g in ((wide[:, :, 3:1603], grad[..., 1:1601]), (wide[:, :, 3:1603].contiguous(), grad[..., 1:1601].contiguous())):
        x = x.detach().requires_grad_(True)
        out = S.short_convolution(x, weight, bias, activation="silu")
        grads = torch.autograd.grad(out, (x, weight), g)
        rows = x.detach().flatten(0, 1) if x.is_contiguous() else wide.flatten(0, 1)[:, 3:1603]
        state, to = torch.zeros(6400, 3, 1600, device=dev), torch.zeros(6400, 1607, dtype=dtype, device=dev)
        with torch.no_grad():
            S.short_convolution_step(rows, state, weight, bias, out=to[:, 5:1605] if not x.is_contiguous() else to[:, :1600])
        results.append((out, *grads, state, to[:, 5:1605] if not x.is_contiguous() else to[:, :1600]))
        outside = to[:, :5] if not x.is_contiguous() else to[:, 1600:]
        assert not outside.any()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def wide_of(t):
    """The same values inside wider rows, at an odd column."""
    big = torch.full((*t.shape[:-1], t.shape[-1] + 5), float("nan"), dtype=t.dtype, device=t.device)
    big[..., 3:3 + t.shape[-1]] = t
    return big[..., 3:3 + t.shape[-1]]


def test_offsets_past_32_bits(dev):
    """Two sequences more than 2^31 elements apart in one buffer."""
    far = 2 ** 31 + 4096
    buf = torch.empty(far + 8192, dtype=torch.bfloat16, device=dev)
    x = buf.as_strided((2, 20, 64), (far, 64, 1))
    x.copy_(torch.randn(2, 20, 64, device=dev))
    dense = x.contiguous()
    w = torch.randn(64, 4, device=dev)
    assert torch.equal(S.short_convolution(x, w), S.short_convolution(dense, w))
    v = some(dev, batch=2, length=20, channels=64, dt=torch.bfloat16)
    call = lambda x: S.state_space_scan(x, v["delta"], v["A"], v["B"], v["C"], gate=x)  # noqa: E731
    assert torch.equal(call(x), call(dense))
    s1, s2 = v["state"].clone(), v["state"].clone()
    step = lambda x, s: S.state_space_step(x, v["delta"][:, 0], s, v["A"], v["B"][:, 0], v["C"][:, 0])  # noqa: E731
    assert torch.equal(step(x[:, 0], s1), step(dense[:, 0], s2)) and torch.equal(s1, s2)
    del buf, x


def test_extreme_step_sizes(dev):
    """delta far below zero leaves the state alone, far above forgets it; infinities are the limits."""
    x = torch.ones(1, 4, 64, device=dev)
    a, b = -torch.ones(64, 4, device=dev), torch.ones(1, 4, 4, device=dev)
    h = torch.full((1, 4, 64), 3.0, device=dev)
    for low in (-200.0, float("-inf")):
        out, last = S.state_space_scan(x, torch.full_like(x, low), a, b, b, state=h, return_state=True)
        assert torch.equal(last, h) and torch.equal(out, torch.full_like(out, 12.0))
    out, last = S.state_space_scan(x, torch.full_like(x, 150.0), a, b, b, state=h, return_state=True)
    assert torch.equal(last, torch.full_like(h, 150.0))
    small = S.state_space_scan(x[:, :1], torch.full_like(x[:, :1], -16.0), a, b[:, :1], b[:, :1] / 4)
    want = torch.log1p(torch.exp(torch.tensor(-16.0, dtype=torch.float64)))
    assert abs(float(small[0, 0, 0]) / float(want) - 1) < 60 * U     # relative: all of the step size's bits are there


def test_saved_tensors_that_move_and_second_derivatives(dev):
    """Packed and unpacked saved tensors (other addresses and strides), checkpointing, and no silent second derivative."""
    v = some(dev, batch=3, length=70, channels=20)
    v["x"] = v["x"].transpose(0, 1).contiguous().transpose(0, 1)
    w, names = torch.randn(20, 4, device=dev), ("x", "delta", "A", "B", "C", "D", "delta_bias", "state")

    def run(leaves):
        u = S.short_convolution(leaves["x"], w, activation="silu")
        return run_scan({**v, **leaves, "x": u})[0]

    def gradients(how):
        leaves = {k: v[k].detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for k in names}
        return torch.autograd.grad(how(leaves).square().sum(), list(leaves.values()))

    want = gradients(run)

    def on_cpu(leaves):
        with torch.autograd.graph.save_on_cpu():
            return run(leaves)

    def checkpointed(leaves):
        return torch.utils.checkpoint.checkpoint(run, leaves, use_reentrant=False)

    def doubled(leaves):   # unpacked beside other values: other strides, perhaps the old address
        with torch.autograd.graph.saved_tensors_hooks(lambda t: torch.stack([t, t], -1).cpu(), lambda t: t.to(dev)[..., 0].contiguous()):
            return run(leaves)

    for how in (on_cpu, checkpointed, doubled):
        assert all(torch.equal(a, b) for a, b in zip(gradients(how), want)), how.__name__
    x = v["x"].clone().requires_grad_(True)
    first, = torch.autograd.grad(S.short_convolution(x, w, activation="silu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiat"):
        torch.autograd.grad(first.sum(), x)


def test_what_is_not_finite_in_a_divided_sequence(dev):
    """A divided sequence hands on what the rows would: zeros through parts that grow past the range, NaN and infinity through parts
    that shrink everything else to nothing, and nothing over a start."""
    gen = torch.Generator().manual_seed(1)
    length, channels, states = 1000, 64, 4
    x, B, C = torch.randn(1, length, channels, generator=gen), torch.randn(1, length, 1, states, generator=gen), torch.randn(1, length, 1, states, generator=gen)
    delta, A = torch.ones(1, length, channels), torch.ones(channels, states) * 4
    x[:, :990] = 0
    on = lambda *t: [v.to(dev) for v in t]  # noqa: E731
    out, last = S.state_space_scan(*on(x, delta, A, B, C), softplus=False, return_state=True)
    want, state = O.state_space_scan(*(t.double() for t in (x, delta, A, B, C)), softplus=False)
    magnitude, state_magnitude = O.state_space_scan(x.double().abs(), delta.double(), A.double(), B.double().abs(), C.double().abs(), softplus=False)
    assert not out[:, :990].any()
    # per row 40 |dt A| + 2 roundings of the decay, ten rows; the sums of 4 terms
    close(out, want, magnitude, 10 * 162 + 10, "out")
    close(last, state, state_magnitude, 10 * 162 + 10, "last")

    starts = torch.zeros(1, length, dtype=torch.bool)
    starts[:, 800] = True
    for value in (float("nan"), float("inf")):
        x = torch.randn(1, length, channels, generator=gen)
        x[0, 10, 7] = value
        got = S.state_space_scan(*on(x, delta, -A, B, C), softplus=False, starts=starts.to(dev)).isfinite().cpu()
        assert not got[0, 10:800, 7].any() and got[0, 800:].all() and got[0, :10].all() and got[..., :7].all() and got[..., 8:].all()


def test_a_directional_difference(dev):
    """The gradient against differences of the kernel's own forward: of a smooth function with terms of order 1 a central
    difference with step 1/64 is off by step^2 / 6 of the third derivative (here under 1e-2) and 2 * rounding / step (1e-4)."""
    v = some(dev, batch=2, length=30, channels=20, states=8)
    torch.manual_seed(0)
    weight = torch.randn(2, 30, 20, device=dev) / 35
    direction = {k: torch.randn_like(t) * 0.1 for k, t in v.items()}
    f = lambda e: float((run_scan({k: t + e * direction[k] for k, t in v.items()})[0].double() * weight).sum())  # noqa: E731
    leaves = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    grads = torch.autograd.grad((run_scan(leaves)[0] * weight).sum(), list(leaves.values()))
    slope = sum(float((g.double() * direction[k]).sum()) for k, g in zip(leaves, grads))
    assert abs((f(1 / 64) - f(-1 / 64)) * 32 - slope) < 1e-2 * max(1.0, abs(slope))


# ---- streams, graphs, command lists ------------------------------------------------------------------------------------
def memory_weights(dev, d, n, seed=9):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen) * scale).to(dev).requires_grad_(True)  # noqa: E731
    return dict(conv=r(d, 4, scale=0.5), conv_bias=r(d, scale=0.1), to_bc=r(d, 2 * n, scale=d ** -0.5), to_delta=r(d, d, scale=0.3 * d ** -0.5),
                delta_bias=(torch.rand(d, generator=gen) * 2 - 4).to(dev).requires_grad_(True),
                A=(-torch.arange(1, n + 1, device=dev).float()).repeat(d, 1).requires_grad_(True), D=r(d), gate=r(d, d, scale=d ** -0.5))


def memory(p, x, states, starts, step):
    """What a recurrent policy does with its features: convolution, projections, recurrence, gate."""
    n = p["A"].shape[1]
    if step:
        u = S.short_convolution_step(x, states[0], p["conv"], p["conv_bias"], activation="silu", starts=starts)
    else:
        u, conv = S.short_convolution(x, p["conv"], p["conv_bias"], activation="silu", state=states[0], starts=starts, return_state=True)
    bc, delta, gate = u @ p["to_bc"], u @ p["to_delta"], x @ p["gate"]
    args = dict(D=p["D"], gate=gate, delta_bias=p["delta_bias"], starts=starts)
    if step:
        return S.state_space_step(u, delta, states[1], p["A"], bc[..., :n], bc[..., n:], **args)
    out, h = S.state_space_scan(u, delta, p["A"], bc[..., :n], bc[..., n:], state=states[1], return_state=True, **args)
    return out, (conv, h)


def test_a_rollout_and_its_training_step(dev):
    """Together as they are used: 24 environment steps with resets, then the recorded rollout at once, whose outputs and
    carried states agree with the steps' and whose gradients agree with the float64 oracle's; then the clip."""
    from isaaclab_amd.utils.gradients import clip_gradient_norm

    envs, steps, d, n = 50, 24, 36, 16
    p = memory_weights(dev, d, n)
    gen = torch.Generator().manual_seed(2)
    obs = torch.randn(steps, envs, d, generator=gen)
    dones = torch.rand(steps, envs, generator=gen) < 0.1
    states0 = (torch.randn(envs, 3, d, generator=gen), torch.randn(envs, n, d, generator=gen))
    states = tuple(s.to(dev) for s in states0)
    outs = []
    with torch.no_grad():
        for t in range(steps):
            outs.append(memory(p, obs[t].to(dev), states, dones[t].to(dev), True))
    starts = dones.to(dev).transpose(0, 1)
    out, last = memory(p, obs.to(dev).transpose(0, 1), tuple(s.to(dev) for s in states0), starts, False)
    torch.testing.assert_close(torch.stack(outs, 1), out.detach(), rtol=2e-4, atol=2e-4)   # two library products in between, in other orders
    torch.testing.assert_close(states[1], last[1].detach(), rtol=2e-4, atol=2e-4)
    torch.testing.assert_close(states[0], last[0].detach(), rtol=0, atol=0)
    loss = out.square().mean()
    loss.backward()
    q = {k: t.detach().cpu().double().requires_grad_(True) for k, t in p.items()}
    x = obs.double().transpose(0, 1)
    u, _ = O.short_convolution(x, q["conv"], q["conv_bias"], True, states0[0].double(), dones.t())
    bc = u @ q["to_bc"]
    ref, _ = O.state_space_scan(u, u @ q["to_delta"], q["A"], bc[..., None, :n], bc[..., None, n:], q["D"], x @ q["gate"], q["delta_bias"], True,
                                states0[1].double(), dones.t())
    ref.square().mean().backward()
    for k in p:
        torch.testing.assert_close(p[k].grad.cpu().double(), q[k].grad, rtol=1e-3, atol=1e-5, msg=lambda m: f"{k}: {m}")
    want = torch.sqrt(sum(g.grad.square().sum() for g in q.values()))
    norm = clip_gradient_norm([t.grad for t in p.values()], float(want) / 2)
    torch.testing.assert_close(norm.cpu().double(), want, rtol=1e-4, atol=0)
    after = torch.sqrt(sum(t.grad.double().square().sum() for t in p.values()))
    torch.testing.assert_close(after.cpu(), want / 2, rtol=1e-4, atol=0)


def test_a_training_step_in_a_graph(dev):
    """Forward and backward captured once and replayed on new inputs, eager work between the replays; two graphs at once."""
    v = some(dev, batch=4, length=50, channels=64)
    w = torch.randn(64, 4, device=dev)

    def train(x, grad):
        x = x.detach().requires_grad_(True)
        u = S.short_convolution(x, w, activation="silu")
        leaves = [x, *(v[k].detach().requires_grad_(True) for k in ("A", "B", "C", "delta"))]
        out = S.state_space_scan(u, leaves[4], *leaves[1:4], D=v["D"], gate=v["gate"], delta_bias=v["delta_bias"], state=v["state"])
        return [out.detach(), *torch.autograd.grad(out, leaves, grad)]

    xs, g = [torch.randn(4, 50, 64, device=dev) for _ in range(3)], torch.randn(4, 50, 64, device=dev)
    want = [[t.clone() for t in train(x, g)] for x in xs]
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        static = xs[0].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            train(static, g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = train(static, g)
        graphs.append((graph, static, result))
    for k in range(4):
        for j, (graph, static, result) in enumerate(graphs):
            i = (k + j) % 3
            static.copy_(xs[i])
            graph.replay()
            eager = train(xs[(i + 1) % 3], g)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(result, want[i])), (k, j)
            assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3]))


def test_parameters_and_a_divided_sequence_in_a_graph(dev):
    """A whole step of parameters' ``.grad``, the way a training loop captures it, with a sequence long enough to be divided."""
    v = some(dev, batch=2, length=300, channels=70)
    names = ("A", "B", "C", "D", "delta_bias")
    x, grad = v["x"].clone(), torch.randn(2, 300, 70, device=dev)
    w = torch.nn.Parameter(torch.randn(70, 4, device=dev))
    p = {k: torch.nn.Parameter(v[k].clone()) for k in names}
    leaves = [w, *p.values()]

    def step():
        u = S.short_convolution(x, w, activation="silu")
        out, _ = run_scan({**v, **p, "x": u})
        out.backward(grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t in leaves:
        t.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    results = [t.grad for t in leaves]
    for k in range(3):
        x.copy_(torch.randn(2, 300, 70, device=dev, generator=torch.Generator(dev).manual_seed(k)))
        for t in leaves:
            t.grad.zero_()
        graph.replay()
        got = [t.clone() for t in results]
        torch.cuda.synchronize()
        eager_x, eager = x.clone(), [t.detach().clone().requires_grad_(True) for t in leaves]
        u = S.short_convolution(eager_x, eager[0], activation="silu")
        out, _ = run_scan({**v, **dict(zip(names, eager[1:])), "x": u})
        want = torch.autograd.grad(out, eager, grad)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_on_another_stream(dev):
    v = some(dev, batch=4, length=600, channels=64)
    want = run_scan(v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run_scan(v) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))


def test_steps_in_a_command_list(dev):
    """A recorded control step, replayed on what its buffers hold; what a list cannot hold is refused."""
    v = some(dev, batch=6, length=8, channels=64)
    w = torch.randn(64, 4, device=dev)
    x, start = torch.zeros(6, 64, device=dev), torch.zeros(6, dtype=torch.bool, device=dev)
    delta, B, C = v["delta"][:, 0].clone(), v["B"][:, 0].clone(), v["C"][:, 0].clone()
    conv, h = torch.zeros(6, 3, 64, device=dev), v["state"].clone()
    commands = CommandList()
    with torch.no_grad(), commands.record():
        u = S.short_convolution_step(x, conv, w, activation="silu", starts=start)
        out = S.state_space_step(u, delta, h, v["A"], B, C, delta_bias=v["delta_bias"], starts=start)
        long, _ = run_scan(v)
    assert len(commands) >= 3
    conv2, h2 = torch.zeros_like(conv), v["state"].clone()
    want_long = run_scan(v)[0]
    for t in range(8):
        x.copy_(v["x"][:, t])
        start.copy_(torch.arange(6, device=dev) == t)
        commands.replay()
        junk = torch.full((1 << 20,), float("nan"), device=dev)  # noqa: F841  (whatever was freed is written over)
        u2 = S.short_convolution_step(x, conv2, w, activation="silu", starts=start)
        out2 = S.state_space_step(u2, delta, h2, v["A"], B, C, delta_bias=v["delta_bias"], starts=start)
        assert torch.equal(out, out2) and torch.equal(conv, conv2) and torch.equal(h, h2) and torch.equal(long, want_long), t
    other = CommandList()
    with other.record():
        with pytest.raises(_abi.IlxError, match="needs gradients"):
            S.short_convolution(v["x"], w.requires_grad_(True))
        with pytest.raises(_abi.IlxError, match="copied"):
            S.state_space_scan(v["x"].transpose(0, 1).contiguous().permute(1, 0, 2), v["delta"], v["A"].t().contiguous().t(), v["B"], v["C"])


# ---- refusals -----------------------------------------------------------------------------------------------------------
def test_refusals(dev):
    x, w = torch.zeros(2, 5, 8, device=dev), torch.zeros(8, 4, device=dev)
    bc, s = torch.zeros(2, 5, 4, device=dev), torch.zeros(2, 4, 8, device=dev)

    def refused(match, call, *args, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            call(*args, **kw)

    conv, scan = S.short_convolution, S.state_space_scan
    refused("batch, length, channels", conv, x[0], w)
    refused("float32, bfloat16 or float16", conv, x.double(), w)
    refused("weight has shape", conv, x, torch.zeros(8, 9, device=dev))
    refused("weight has shape", conv, x, torch.zeros(7, 4, device=dev))
    refused("parameters and states are float32", conv, x, w.half())
    refused("activation", conv, x, w, activation="relu")
    refused("bias has shape", conv, x, w, w[:, :1])
    refused("state has shape", conv, x, w, state=s)
    refused("starts", conv, x, w, starts=torch.zeros(2, 4, dtype=torch.bool, device=dev))
    refused("starts", conv, x, w, starts=torch.zeros(2, 5, device=dev))
    refused("lengths", conv, x, w, lengths=torch.zeros(2, device=dev))
    refused("lengths is on", conv, x, w, lengths=torch.zeros(2, dtype=torch.int32))
    refused("weight is on", conv, x, w.cpu())
    refused("no channels", conv, x[..., :0], w[:0])
    refused("delta has shape", scan, x, x[:, :4], w, bc, bc)
    refused("delta is", scan, x, x.half(), w, bc, bc)
    refused("A has shape", scan, x, x, torch.zeros(8, 33, device=dev), bc, bc)
    refused("B has shape", scan, x, x, w, bc[:, :4], bc)
    refused("4 states", scan, x, x, w, bc[..., :3], bc[..., :3])
    refused("groups", scan, x, x, w, bc[:, :, None].expand(2, 5, 3, 4), bc[:, :, None].expand(2, 5, 3, 4))
    refused("C is", scan, x, x, w, bc, bc.half())
    refused("gate has shape", scan, x, x, w, bc, bc, gate=x[..., :4])
    refused("D has shape", scan, x, x, w, bc, bc, D=w)
    step = S.short_convolution_step
    refused("carried state", step, x[:, 0], None, w)
    refused("contiguous", step, x[:, 0], torch.zeros(2, 8, 3, device=dev).transpose(1, 2), w)
    refused("out must", step, x[:, 0], torch.zeros(2, 3, 8, device=dev), w, out=x[:, 0].half())
    refused("overlap", step, x[:, 0], torch.zeros(2, 3, 8, device=dev), w, out=torch.zeros(8, device=dev).expand(2, 8))
    refused("no backward", step, x[:, 0], torch.zeros(2, 3, 8, device=dev), w.clone().requires_grad_(True), error=RuntimeError)
    refused("no backward", S.state_space_step, x[:, 0], x[:, 0], s.clone().requires_grad_(True), w, bc[:, 0], bc[:, 0], error=RuntimeError)
    # a state that a backward pass still needs is not silently the wrong one
    weight, state = w.clone().requires_grad_(True), torch.zeros(2, 3, 8, device=dev)
    out = conv(x, weight, state=state)
    with torch.no_grad():
        step(x[:, 0], state, weight)
    refused("modified by an inplace", torch.autograd.grad, out.sum(), weight, error=RuntimeError)
