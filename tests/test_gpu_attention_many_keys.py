"""GPU: one key that takes most of a row's weight beside many thousands of keys that share the rest.
Each of those is far below the row's largest probability, and together they are part of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [65536, 20011])
@pytest.mark.parametrize("gap", [15.0, 22.6, 25.1, 28.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_dominant_key(cuda_lib, dtype, gap, n):
    """Every query meets key 0 with a score `gap` powers of two above all others.

    Bounds (h half a step of the type, t = 2e-5 for the 32-bit sums and exponentials): out
    h (|o| + P|V|) + t P|V|, and for fp16 the smallest steps: P holds 2^7 exp(s - max) or more, so a key
    below the normal range loses up to 2^-25 / 2^7 of the row's largest probability, and the output itself
    up to 2^-25.  dq: the same loss of o in do.o (the output's own rounding is kept beside it), ds rounded
    once, and fp16's smallest steps again: ds is scaled so that the largest |dO||V| + |delta| is at least
    2^14 (M 2^-39 each), P with 2^8 (2^-33 each, times dP - delta)."""
    from stew_b200.step_ops import packed_attention
    d, scale = 64, 1.0
    g = torch.Generator(device="cuda").manual_seed(n)
    q = torch.zeros(n, 1, d, device="cuda")
    q[..., 0] = 4.0
    k = torch.randn(n, 1, d, device="cuda", generator=g)
    k[..., 0] = 0.0
    k[0, 0, 0] = gap * math.log(2.0) / 4.0
    v = -1.0 - torch.rand(n, 1, d, device="cuda", generator=g)
    v[0] = 1.0
    dout = torch.randn(n, 1, d, device="cuda", generator=g) * 0.02
    q, k, v, dout = (x.to(dtype) for x in (q, k, v, dout))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*leaves, cu, window=(-1, -1), scale=scale)
    (dq,) = torch.autograd.grad(out, leaves[:1], dout)

    rows = torch.tensor([0, 1, 63, 64, 1000, n // 2, n - 1], device="cuda")
    Q, K, V, dO = (x.detach()[:, 0].double() for x in (q, k, v, dout))
    Q, dO = Q[rows], dO[rows]
    p = torch.softmax(scale * Q @ K.T, -1)
    o, pv = p @ V, p @ V.abs()
    h, t = torch.finfo(dtype).eps / 2, 2e-5
    half = dtype == torch.float16
    top = p.amax(-1, keepdim=True)
    lost = 2.0 ** -32 * top * V.abs().sum(0) if half else torch.zeros_like(o)
    bound = h * (o.abs() + pv) + t * pv + lost + (2.0 ** -25 if half else 0.0)
    err = (out.detach()[rows, 0].double() - o).abs()
    assert bool((err <= 1.05 * bound).all()), float((err / bound).max())
    # the weight of the many keys, free of P's rounding: all of them hold one value
    weight = float(1 - p[0, 0])
    assert weight > 2.0 ** -25 * n / 8

    dp = dO @ V.T
    delta = (dO * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    eo = h * pv + t * pv + lost  # of the forward's sum
    edelta = (dO.abs() * eo).sum(-1, keepdim=True)
    eds = h * ds.abs() + p * edelta + t * p * (dO.abs() @ V.abs().T + (dO.abs() * o.abs()).sum(-1, keepdim=True))
    if half:
        size = dout.double().norm(dim=2).max() * V.norm(dim=1).max() + (dout.double() * out.double()).sum(2).abs().max()
        eds = eds + size * 2.0 ** -39
    ref = scale * ds @ K
    bound = scale * eds @ K.abs() + h * ref.abs() + (2.0 ** -25 if half else 0.0)
    err = (dq[rows, 0].double() - ref).abs()
    assert bool((err <= 1.05 * bound).all()), float((err / bound).max())


@pytest.mark.parametrize("scale", [1.0, 6.0])
def test_log_sum_exp_is_unscaled(cuda_lib, scale):
    """The saved log-sum-exp is the definition's whatever factor P carries: fp32 rounding of a maximum up
    to ~60 and of the sums (2e-5)."""
    from stew_b200.step_ops import _attn_forward
    g = torch.Generator(device="cuda").manual_seed(3)
    for dtype in (torch.float16, torch.bfloat16):
        q, k, v = (torch.randn(300, 2, 64, device="cuda", generator=g).to(dtype) for _ in range(3))
        cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
        lse = _attn_forward(q, k, v, cu, -1, -1, scale)[2]
        s = scale * torch.einsum("ihd,jhd->hij", q.double(), k.double())
        want = torch.logsumexp(s, -1)
        assert bool(((lse.double() - want).abs() <= 2e-5 + 4 * 2.0 ** -24 * want.abs()).all())
