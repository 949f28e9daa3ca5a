"""GPU: gradient norm and clipping where lists and tensors outgrow one launch's table and one share a workgroup.

Bounds as in tests/test_gradients_gpu.py: the norm is off by 2 u (u = 2^-24), a scaled gradient by 5 u and half a step of its type."""

import math

import pytest
import torch

from isaaclab_amd.utils.gradients import clip_gradient_norm, gradient_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
M = 1 << 20


def make(dev, sizes, dtypes):
    gen = torch.Generator(dev).manual_seed(len(sizes))
    return [torch.randn(n, generator=gen, device=dev).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def norm64(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


@pytest.mark.parametrize("name,sizes,dtypes", [
    ("one table, full", [5 + i % 300 for i in range(223)], ["float32", "bfloat16"]),
    ("one more", [5 + i % 300 for i in range(224)], ["float32", "bfloat16"]),
    ("two tables", [1 + (i * 53) % 2000 for i in range(301)], ["bfloat16", "float16", "float32"]),
    ("two tables, empty ones between", [(i % 3) * 97 for i in range(640)], ["float32"]),
    ("five tables", [11 + i % 7 for i in range(1000)], ["float16"]),
    ("more shares than workgroups in both launches", [70 * M + 13, 5, M + 1], ["bfloat16"]),
    ("many shares in two tables", [3000] * 230 + [40 * M + 7, 40 * M + 1] + [3000] * 50, ["bfloat16", "float32"]),
])
def test_norm_and_clip(dev, name, sizes, dtypes):
    grads = make(dev, sizes, [getattr(torch, d) for d in dtypes])
    before = [g.clone() for g in grads]
    want = norm64(grads)
    assert abs(float(gradient_norm(grads)) - want) <= 2 * U * want
    most = max(float(g.abs().max()) for g in grads if g.numel())
    assert float(gradient_norm(grads, math.inf)) == most
    assert abs(float(clip_gradient_norm(grads, want * 1.01)) - want) <= 2 * U * want
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    bound = float(torch.tensor(want * 0.3))
    assert abs(float(clip_gradient_norm(grads, bound)) - want) <= 2 * U * want
    for i, (g, b) in enumerate(zip(grads, before)):
        expect = b.double() * (bound / (want + 1e-6))
        half = 0.0 if g.dtype == torch.float32 else torch.finfo(g.dtype).eps / 2
        limit = expect.abs() * (5 * U + half) * (1 + 2 * half) + (2.0 ** -25 if g.dtype == torch.float16 else 1e-45)
        assert ((g.double() - expect).abs() <= limit).all(), i


def test_a_tensor_of_several_table_entries(dev):
    """More than 2^30 elements: ones, whose norm is the root of their number and whose scaled value is one number."""
    n = (1 << 30) + 20001
    grads = [torch.ones(3, device=dev), torch.ones(n, dtype=torch.bfloat16, device=dev)]
    want = math.sqrt(n + 3)
    norm = clip_gradient_norm(grads, want / 4)
    assert abs(float(norm) - want) <= 2 * U * want
    assert bool((grads[1] == 0.25).all()) and ((grads[0] - 0.25).abs() <= 5 * U).all()


def test_a_scaled_tensor_of_few_shares_beside_many(dev):
    """The elements around the border of every share are scaled once: marks there, in one tensor and across tensors."""
    sizes = [16384 * 3, 16385, 16383, 1, 16384]
    grads = [torch.arange(1, n + 1, device=dev, dtype=torch.float32) for n in sizes]
    before = [g.clone() for g in grads]
    want = norm64(grads)
    clip_gradient_norm(grads, want / 2)
    for g, b in zip(grads, before):
        assert ((g.double() / b.double() - 0.5).abs() <= 5 * U).all()
