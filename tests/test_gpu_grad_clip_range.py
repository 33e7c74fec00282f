"""GPU: clipping whose factor is outside fp32's normal range, while the results are inside: the factor
max_norm / norm of very large gradients and a small limit, the reciprocal of a very small divisor."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def _grads(dtype, scale, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, device="cuda", generator=g, dtype=torch.float64) * scale).to(dtype) for n in (5000, 3, 1, 4099)]


def _check(grads, max_norm, div, out):
    from stew_b200.dp import clip_grads
    d = 1.0 if div is None else float(torch.tensor(div, dtype=torch.float32))
    limit = float(torch.tensor(max_norm, dtype=torch.float32))
    src = [g.double() for g in grads]
    norm = math.sqrt(sum(float(g.square().sum()) for g in src)) / abs(d)
    c = min(1.0, limit / (norm + 1e-6))
    dst = [torch.empty_like(g) for g in grads] if out else grads
    got = clip_grads(grads, max_norm, divisor=None if div is None else torch.tensor([div], device="cuda"),
                     out=dst if out else None)
    if norm < 3e38:
        assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for g, s in zip(dst, src):
        want = s / d * c
        h = torch.finfo(g.dtype).eps / 2  # and the factor's rounding and the product's, as in the normal range
        err = (g.double() - want).abs()
        assert bool((err <= (h + 3 * 2.0 ** -24) * want.abs() + TINY[g.dtype]).all()), float(err.max())


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale,max_norm", [(1e30, 1e-10), (1e33, 1e-16), (1e36, 1e-3), (1e30, 1e-20), (3e37, 1.0)])
def test_factor_below_the_normal_range(cuda_lib, dtype, scale, max_norm, out):
    _check(_grads(dtype, scale), max_norm, None, out)


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale,div,max_norm", [(1e-30, 1e-39, math.inf), (1e-37, 3e-40, 1e6), (1e-30, 1e-45, 1e30),
                                                (1e30, 1e38, 1e-15), (1e-30, -1e-39, math.inf)])
def test_divisors_outside_the_normal_range(cuda_lib, dtype, scale, div, max_norm, out):
    _check(_grads(dtype, scale), max_norm, div, out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_limit_zero_gives_zeros(cuda_lib, dtype):
    from stew_b200.dp import clip_grads
    grads = _grads(dtype, 1.0)
    clip_grads(grads, 0.0)
    assert not any(bool(g.any()) for g in grads)
