"""GPU: global gradient norm and clipping (nf4b_clip_grads, dp.clip_grads) against 64-bit torch.
Bounds: the norm is a 64-bit sum rounded once to fp32 (2^-24 relative; 1e-6 + eps in the factor);
a result is src times an fp32 factor: the factor's rounding and the product's, 2 x 2^-24
relative, then the type's own half step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _grads(sizes, dtype, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * scale).to(dtype) for s in sizes]


def _reference(grads, max_norm, div=1.0):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads)) / abs(div)
    c = min(1.0, max_norm / (norm + 1e-6))
    return norm, [g.double() / div * c for g in grads]


def _close(got, want):
    h = torch.finfo(got.dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[got.dtype]
    err = (got.double() - want).abs()
    assert bool((err <= (h + 3 * 2.0 ** -24) * want.abs() + tiny).all()), float((err / want.abs().clamp_min(1e-300)).max())


SIZES = [[1], [7], [4096], [4097, 3, 0, 1], [16 * 1536, 1536 * 16, 16 * 1536, 256 * 16] * 28, [100003, 5, 64, 8191],
         [33] * 1200, [(1 << 20) + 5]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("max_norm,div", [(0.5, None), (1e9, None), (2.0, 37.0)])
def test_norm_and_clip_in_place(cuda_lib, dtype, sizes, max_norm, div):
    from stew_b200.dp import clip_grads
    grads = _grads(sizes, dtype)
    norm, want = _reference(grads, max_norm, div or 1.0)
    before = [g.clone() for g in grads]
    got = clip_grads(grads, max_norm, divisor=None if div is None else torch.tensor([div], device="cuda"))
    assert got.shape == () and abs(float(got) - norm) <= 2.0 ** -23 * norm
    for g, w in zip(grads, want):
        _close(g, w)
    if norm < max_norm and div is None:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("dtype", TYPES)
def test_out_of_place_from_a_flat_buffer(cuda_lib, dtype):
    """Views at odd offsets of a flat buffer (2- or 4-byte aligned only) into tensors of their own:
    the inputs stay, the gaps of the buffers stay."""
    from stew_b200.dp import clip_grads
    sizes = [1, 6, 333, 4095, 4096, 4099, 20000]
    flat = _grads([sum(sizes) + 1], dtype)[0]
    keep = flat.clone()
    src = list(flat[1:].split(sizes))
    out = torch.full((sum(sizes) + 2 * len(sizes),), 7.0, device="cuda").to(dtype)
    dst, at = [], 1
    for s in sizes:
        dst.append(out[at:at + s])
        at += s + 2
    norm, want = _reference(src, 1.0, 8.0)
    got = clip_grads(src, 1.0, divisor=torch.tensor([8.0], device="cuda"), out=dst)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm and torch.equal(flat, keep)
    for d, w in zip(dst, want):
        _close(d, w)
    mask = torch.ones_like(out, dtype=torch.bool)
    at = 1
    for s in sizes:
        mask[at:at + s] = False
        at += s + 2
    assert bool((out[mask] == 7.0).all())


def test_mixed_types_in_one_list(cuda_lib):
    from stew_b200.dp import clip_grads
    grads = [t for d in TYPES for t in _grads([1000, 77], d)]
    norm, want = _reference(grads, 3.0)
    assert abs(float(clip_grads(grads, 3.0)) - norm) <= 2.0 ** -23 * norm
    for g, w in zip(grads, want):
        _close(g, w)


@pytest.mark.parametrize("scale", [1e-30, 1e25])
def test_squares_outside_fp32(cuda_lib, scale):
    from stew_b200.dp import clip_grads
    for dtype in (torch.float32, torch.bfloat16):
        grads = _grads([5000, 3], dtype, scale)
        norm, want = _reference(grads, 1.0)
        assert abs(float(clip_grads(grads, 1.0)) - norm) <= 2.0 ** -23 * norm
        for g, w in zip(grads, want):
            _close(g, w)


def test_not_finite(cuda_lib):
    from stew_b200.dp import clip_grads
    g = [torch.tensor([1.0, float("inf"), -2.0], device="cuda"), torch.ones(5, device="cuda")]
    assert math.isinf(float(clip_grads(g, 1.0)))
    assert torch.isnan(g[0][1]) and not g[0][[0, 2]].any() and not g[1].any()
    g = [torch.tensor([1.0, float("nan")], device="cuda"), torch.ones(5, device="cuda")]
    assert math.isnan(float(clip_grads(g, 1.0)))
    assert torch.isnan(g[0]).all() and torch.isnan(g[1]).all()
    g = [torch.tensor([1.0, float("inf")], device="cuda")]
    assert math.isinf(float(clip_grads(g, math.inf))) and torch.isnan(g[0]).all()
    z = [torch.zeros(9, device="cuda")]
    assert float(clip_grads(z, 1.0)) == 0.0 and not z[0].any()
    z = [torch.ones(9, device="cuda")]
    assert float(clip_grads(z, math.inf)) == 3.0 and bool((z[0] == 1).all())
    assert float(clip_grads(z, 0.0)) == 3.0 and not z[0].any()
    assert float(clip_grads([torch.empty(0, device="cuda")], 1.0)) == 0.0


def test_autograd_notices_the_write(cuda_lib):
    """A gradient that an autograd graph saved and clip_grads then scaled ends that graph's backward
    with torch's error; out of place only the outputs count as written."""
    from stew_b200.dp import clip_grads
    for out in (False, True):
        g, a = torch.full((9,), 3.0, device="cuda"), torch.ones(9, device="cuda", requires_grad=True)
        y = (a * g).sum()
        clip_grads([g], 1.0, out=[torch.empty_like(g)] if out else None)
        if out:
            assert torch.equal(torch.autograd.grad(y, a)[0], g)
        else:
            with pytest.raises(RuntimeError, match="inplace operation"):
                y.backward()


def test_same_bits_and_matches_torch(cuda_lib):
    from stew_b200.dp import clip_grads
    sizes = [24576, 24576, 24576, 4096] * 28
    runs = []
    for _ in range(4):
        grads = _grads(sizes, torch.float32)
        n = clip_grads(grads, 1.0)
        runs.append([n] + grads)
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
    params = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in sizes]
    for p, g in zip(params, _grads(sizes, torch.float32)):
        p.grad = g
    ref = torch.nn.utils.clip_grad_norm_(params, 1.0)
    assert abs(float(ref) - float(runs[0][0])) <= 1e-5 * float(ref)
    for p, g in zip(params, runs[0][1:]):
        assert torch.allclose(p.grad, g, rtol=1e-5, atol=0)


def test_captured_and_replayed(cuda_lib):
    """Two captured graphs and an eager call, replayed in turn: none sees another's scratch."""
    from stew_b200.dp import clip_grads
    sets = [_grads([3000, 50], torch.float32, seed=s) for s in (1, 2)]
    outs = [[torch.empty_like(g) for g in s] for s in sets]
    graphs, norms = [], []
    for s, o in zip(sets, outs):
        clip_grads(s, 1.0, out=o)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(clip_grads(s, 1.0, out=o))
        graphs.append(g)
    for _ in range(2):
        for s in sets:
            for t in s:
                t.mul_(1.5)
        for g in graphs:
            g.replay()
        for s, o, n in zip(sets, outs, norms):
            norm, want = _reference(s, 1.0)
            assert abs(float(n) - norm) <= 2.0 ** -23 * norm
            for a, b in zip(o, want):
                _close(a, b)


def test_past_32_bit_counts(cuda_lib):
    """One tensor of more than 2^31 values."""
    from stew_b200.dp import clip_grads
    n = (1 << 31) + 4099
    g = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    norm = clip_grads([g], 1.0)
    assert abs(float(norm) - math.sqrt(n)) <= 2.0 ** -23 * math.sqrt(n)
    want = torch.tensor(1.0 / math.sqrt(n)).bfloat16().cuda()
    assert bool((g[:4096] == want).all()) and bool((g[-5000:] == want).all()) and bool((g[1 << 30] == want))
