"""The norm of all gradients and their clipping against 64 bits, on the GPU."""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_fp8 import HALF, SMALL

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _grads(g, sizes, dtype, scale=1.0):
    return [(torch.randn(s, generator=g, device="cuda") * scale * (1 + i)).to(dtype) for i, s in enumerate(sizes)]


def _norm(grads):
    return math.sqrt(sum(float(x.double().square().sum()) for x in grads))


def check(out, grads, norm, max_norm):
    want = _norm(grads)
    assert abs(float(norm) - want) <= want * 2.0 ** -23
    f = max_norm / want if want > max_norm else 1.0
    for o, x in zip(out, grads):
        w = x.double() * f
        assert bool(((o.double() - w).abs() <= w.abs() * (2.0 ** -23 + HALF[o.dtype] * 1.001) + SMALL[o.dtype]).all())


SIZES = [[1], [(3, 5)], [8192], [8193, 7], [(64, 64)] * 49, [1] * 100, [(1000, 1000), 17, (33, 3, 5), 0, 8191], [3_000_001]]


@pytest.mark.parametrize("sizes", SIZES, ids=range(len(SIZES)))
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_clipping(cuda, sizes, dtype):
    from engraft_ngram_amd import clip
    grads = _grads(_gen(len(sizes)), sizes, dtype)
    want = _norm(grads)
    kept = [x.clone() for x in grads]
    assert abs(float(clip.grad_norm(grads)) - want) <= want * 2.0 ** -23
    for max_norm in (want * 0.3, want * 1.5):
        for out_dtype in (dtype, F32):
            out = [torch.full(x.shape, float("nan"), dtype=out_dtype, device="cuda") for x in grads]
            n = clip.clip_grads(grads, max_norm, out=out)
            check(out, grads, n, max_norm)
            assert all(torch.equal(a, b) for a, b in zip(grads, kept))
            again = [torch.empty_like(x) for x in out]
            assert torch.equal(n, clip.clip_grads(grads, max_norm, out=again)) and all(torch.equal(a, b) for a, b in zip(out, again))
        versions = [x._version for x in grads]
        in_place = [x.clone() for x in grads]
        clip.clip_grads(in_place, max_norm)
        out = [torch.empty_like(x) for x in grads]
        clip.clip_grads(grads, max_norm, out=out)
        assert all(torch.equal(a, b) for a, b in zip(in_place, out))
        assert [x._version for x in grads] == versions and all(x._version > 0 for x in in_place)
    assert float(clip.clip_grads(in_place, 0.0)) >= 0 and not any(bool(x.any()) for x in in_place)


def test_sums_of_the_largest_and_smallest(cuda):
    """Squares past the largest fp32 number and below the smallest; a factor below the normal numbers."""
    from engraft_ngram_amd import clip
    big, small = torch.full((5000,), 3e38, device="cuda"), torch.full((5000,), 1e-40, device="cuda")
    assert float(clip.grad_norm([small])) == pytest.approx(1e-40 * math.sqrt(5000), rel=1e-4)
    assert math.isinf(float(clip.grad_norm([big])))  # the sum is finite, its root is no fp32 number
    out = [torch.empty_like(big)]
    clip.clip_grads([big], 1.0, out=out)
    assert bool(((out[0].double() * math.sqrt(5000) - 1.0).abs() < 1e-6).all())
    out = [torch.empty_like(big)]
    clip.clip_grads([big], 1e-6, out=out)
    assert bool(((out[0].double() * math.sqrt(5000) * 1e6 - 1.0).abs() < 1e-6).all())


def test_a_norm_that_is_not_finite_leaves_the_values(cuda):
    from engraft_ngram_amd import clip
    for bad in (float("nan"), float("inf")):
        grads = _grads(_gen(2), [100, 9000], F32)
        grads[1][77] = bad
        kept = [x.clone() for x in grads]
        n = clip.clip_grads(grads, 1e-3)
        assert not math.isfinite(float(n))
        assert all(torch.equal(torch.nan_to_num(a, nan=5.5), torch.nan_to_num(b, nan=5.5)) for a, b in zip(grads, kept))


def test_a_tensor_past_4_gib(cuda):
    from engraft_ngram_amd import clip
    x = torch.zeros((1 << 31) + 5, dtype=BF16, device="cuda")
    x[-3:] = torch.tensor([3.0, -4.0, 12.0])
    x[0] = 84.0
    assert float(clip.clip_grads([x], 8.5)) == 85.0
    assert x[-3:].tolist() == [0.30078125, -0.400390625, 1.203125] and float(x[0]) == 8.375  # the nearest bf16 to 0.3, 0.4, 1.2, 8.4
    assert float(x[1:-3].abs().max()) == 0.0


def test_strides(cuda):
    """Rows of wider buffers, transposes, mixed types; what lies between the rows stays."""
    from engraft_ngram_amd import clip
    g = _gen(3)
    wide = torch.randn((300, 90), generator=g, device="cuda")
    kept = wide.clone()
    a, b = wide[:, 5:42], wide[:, 50:77]
    t = torch.randn((40, 60), generator=g, device="cuda").to(BF16).T
    h = torch.randn((7, 8, 9), generator=g, device="cuda").to(F16)
    grads = [a, b, t, h]
    before = [x.clone() for x in grads]
    n = clip.clip_grads(grads, 2.0)
    check(grads, before, n, 2.0)
    gap = torch.ones(90, dtype=torch.bool, device="cuda")
    gap[5:42] = gap[50:77] = False
    assert torch.equal(wide[:, gap], kept[:, gap])
    # into outputs of other strides
    out = [torch.empty((300, 37), device="cuda"), torch.empty((27, 300), device="cuda")]
    with pytest.raises(ValueError):
        clip.clip_grads([a, b], 1.0, out=[out[0], out[1].T])
    out[1] = torch.empty((300, 200), device="cuda")[:, 100:127]
    before = [a.clone(), b.clone()]
    check(out, before, clip.clip_grads([a, b], 1.0, out=out), 1.0)
    plain = torch.randn((300, 27), generator=g, device="cuda")
    check([out[1]], [plain], clip.clip_grads([plain], 1.0, out=[out[1]]), 1.0)


def test_graphs_and_streams(cuda):
    from engraft_ngram_amd import clip
    g = _gen(4)
    grads = _grads(g, [10_000, (30, 40), 5], F32)
    out = [torch.empty_like(x) for x in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = clip.clip_grads(grads, 1.0, out=out)
    for k in range(3):
        for x in grads:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda") * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        check(out, grads, n, 1.0)
        eager = [torch.empty_like(x) for x in grads]
        assert torch.equal(n, clip.clip_grads(grads, 1.0, out=eager)) and all(torch.equal(a, b) for a, b in zip(out, eager))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        m = clip.grad_norm(grads)
    side.synchronize()
    assert torch.equal(m, n)
