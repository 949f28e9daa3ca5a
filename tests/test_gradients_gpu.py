"""GPU: global gradient norm and clipping against float64.

The squares are added in 64 bits, so the norm is off by the rounding to float32, u = 2^-24 relative (2 u with the 64-bit sums of
either side); the factor min(1, max_norm (1 / (norm + 1e-6))) adds three roundings and the product one, 5 u in all, and a 16-bit
gradient is rounded once more, by at most half a step of its type."""

import math

import pytest
import torch

from isaaclab_amd.utils.command_list import CommandList
from isaaclab_amd.utils.gradients import clip_gradient_norm, gradient_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = {
    "one": [1],
    "scalars": [1, 1, 1],
    "odd": [3, 17, 1, 255, 4097, 16384, 16385, 7],
    "empty": [0, 5, 0, 0, 12, 0],
    "only empty": [0, 0],
    "policy": [235 * 512, 512, 512 * 256, 256, 256 * 128, 128, 128 * 12, 12],
    "two tables": [10 + i % 7 for i in range(97)],
    "many": [1 + (i * 37) % 400 for i in range(500)],
    "large": [3_000_001, 77],
}


def make(dev, sizes, dtypes, scale=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * scale).to(dtypes[i % len(dtypes)]).to(dev) for i, n in enumerate(sizes)]


def norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check_scaled(grads, before, coef):
    for i, (g, b) in enumerate(zip(grads, before)):
        want = b.double() * coef
        half = 0.0 if g.dtype == torch.float32 else torch.finfo(g.dtype).eps / 2
        bound = want.abs() * (5 * U + half) * (1 + 2 * half) + (0 if g.dtype != torch.float16 else 2.0 ** -25) + 1e-45
        assert ((g.double() - want).abs() <= bound).all(), i


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16, torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("name", SIZES)
def test_norm_and_clip(dev, name, dtypes):
    grads = make(dev, SIZES[name], dtypes)
    before = [g.clone() for g in grads]
    want = norm64(before)
    got = gradient_norm(grads)
    assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - want) <= 2 * U * want
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    most = max((float(g.double().abs().max()) for g in before if g.numel()), default=0.0)
    assert float(gradient_norm(grads, math.inf)) == most
    assert float(clip_gradient_norm(grads, want * 1.01 + 1e-3)) == float(got)
    assert all(torch.equal(a, b) for a, b in zip(grads, before)), "a norm below the bound changes nothing"
    assert float(clip_gradient_norm(grads, want * 0.3)) == float(got)
    check_scaled(grads, before, min(1.0, float(torch.tensor(want * 0.3).float()) / (want + 1e-6)))
    grads = [b.clone() for b in before]
    assert float(clip_gradient_norm(grads, 0.5, math.inf)) == most
    check_scaled(grads, before, min(1.0, 0.5 / (most + 1e-6)))


def test_alignment_and_layout(dev):
    """Views at any element of a flat buffer, and dense tensors in another order of dimensions."""
    flat = make(dev, [10_000], [torch.bfloat16])[0]
    grads = [flat[1:1000], flat[1003:1004], flat[1005:1012], flat[2001:9999], torch.randn(6, 5, 4, device=dev).permute(2, 0, 1),
             torch.randn(3, 4, device=dev).t()]
    keep, outside = [g.clone() for g in grads], flat.clone()
    clip_gradient_norm(grads, 1.0)
    check_scaled(grads, keep, 1.0 / (norm64(keep) + 1e-6))
    for at in (0, 1000, 1002, 1004, 1012, 2000, 9999):
        assert flat[at] == outside[at]


def test_range(dev):
    """Squares past float32's range count; zeros stay zeros; none of the factors is a NaN by accident."""
    grads = [torch.full((100,), 1e30, device=dev), torch.full((5,), 1e-30, device=dev)]
    norm = clip_gradient_norm(grads, 1.0)
    assert abs(float(norm) / 1e31 - 1) < 4 * U
    torch.testing.assert_close(grads[0], torch.full((100,), 0.1, device=dev), rtol=1e-6, atol=0)
    small = [torch.full((4,), 1e-30, device=dev)]
    assert abs(float(gradient_norm(small)) / 2e-30 - 1) < 4 * U
    zeros = [torch.zeros(9, device=dev)]
    assert float(clip_gradient_norm(zeros, 0.0)) == 0.0 and not zeros[0].any()
    some = [torch.ones(9, device=dev)]
    clip_gradient_norm(some, 0.0)
    assert not some[0].any()
    some = [torch.ones(9, device=dev)]
    clip_gradient_norm(some, math.inf)
    assert torch.equal(some[0], torch.ones(9, device=dev))


def test_not_finite(dev):
    one = lambda *v: [torch.tensor(v, device=dev), torch.ones(3, device=dev)]  # noqa: E731
    for kind in (2.0, math.inf):
        g = one(float("inf"), 1.0)
        assert float(clip_gradient_norm(g, 1.0, kind)) == math.inf
        assert torch.isnan(g[0][0]) and g[0][1] == 0 and not g[1].any()
        g = one(float("nan"), 1.0)
        assert math.isnan(float(clip_gradient_norm(g, 1.0, kind))) and torch.isnan(g[0]).all() and torch.isnan(g[1]).all()
        assert math.isnan(float(gradient_norm(one(float("nan"), float("inf")), kind)))
        assert float(gradient_norm(one(float("-inf"), 1.0), kind)) == math.inf


def test_graph_and_command_list(dev):
    base = make(dev, SIZES["many"], [torch.float32, torch.bfloat16])
    grads = [b.clone() for b in base]
    clip_gradient_norm(grads, 1.0)
    want = [g.clone() for g in grads]
    commands, graph = CommandList(), torch.cuda.CUDAGraph()
    with commands.record():
        norm = clip_gradient_norm(grads, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph):
        norm_graph = clip_gradient_norm(grads, 1.0)
    for k in range(6):
        for g, b in zip(grads, base):
            g.copy_(b)
        commands.replay() if k % 2 else graph.replay()
        junk = torch.full((1 << 16,), float("nan"), device=dev)  # noqa: F841
        gradient_norm(base)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want)), k
        assert abs(float(norm if k % 2 else norm_graph) - norm64(base)) <= 2 * U * norm64(base)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rounds_as_torch_does(dev, dtype):
    """The scale has the bits of torch's ``max_norm / (norm + 1e-6)`` in float32, so no 16-bit gradient rounds another way."""
    for seed in range(8):
        grads = make(dev, [50_001, 300], [dtype], seed=seed)
        before = [g.clone() for g in grads]
        norm = clip_gradient_norm(grads, 7.3 + seed)
        scale = torch.clamp((7.3 + seed) / (norm + 1e-6), max=1.0)
        assert all(torch.equal(g, (b.float() * scale).to(dtype)) for g, b in zip(grads, before))


def test_two_runs_agree_bit_for_bit(dev):
    grads = make(dev, [5_000_000, 123_457], [torch.float32])
    assert len({float(gradient_norm(grads)) for _ in range(5)}) == 1


def test_refusals(dev):
    g = torch.ones(8, device=dev)
    for match, call in (
            ("no gradients", lambda: clip_gradient_norm([None], 1.0)),
            ("max_norm", lambda: clip_gradient_norm([g], -1.0)),
            ("max_norm", lambda: clip_gradient_norm([g], math.nan)),
            ("norm_type", lambda: gradient_norm([g], 1.0)),
            ("float32, bfloat16 or float16", lambda: gradient_norm([g.double()])),
            ("not dense", lambda: clip_gradient_norm([torch.ones(8, 8, device=dev)[:, ::2]], 1.0)),
            ("not dense", lambda: clip_gradient_norm([g[:1].expand(4)], 1.0)),
            ("is on", lambda: clip_gradient_norm([g, g.cpu()], 1.0)),
            ("share memory", lambda: clip_gradient_norm([g, g], 1.0)),
            ("share memory", lambda: clip_gradient_norm([g[4:], g[:5]], 1.0))):
        with pytest.raises((ValueError, RuntimeError), match=match):
            call()
    assert torch.equal(g, torch.ones(8, device=dev))
    assert abs(float(gradient_norm([g, g])) - 4.0) < 1e-6     # a norm alone may count a tensor twice
