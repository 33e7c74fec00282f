"""GPU: how exact a sequence's gradients are does not depend on what is packed beside it."""
import math

import pytest
import torch

from tests.attention_ref import reference

pytestmark = pytest.mark.gpu


def _inputs(lens, dtype, d, pad=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    edges = [0]
    for x in lens:
        edges.append(edges[-1] + x)
    n = edges[-1]
    q, k, v, dout = (torch.randn(n, h, d, device="cuda", generator=g) for h in (4, 2, 2, 4))
    dout *= 0.02
    more = lambda t: torch.cat([t, torch.ones(pad, *t.shape[1:], device="cuda")]).to(dtype)
    return [more(t) for t in (q, k, v)], torch.tensor(edges, dtype=torch.int32, device="cuda"), edges, more(dout)


def _grads(leaves, cu, dout):
    from stew_b200.step_ops import packed_attention
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    return torch.autograd.grad(packed_attention(*leaves, cu), leaves, dout)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[4000] + [2] * 40, [3, 2, 2, 5, 4, 9] * 8 + [20000], [1500, 100, 1, 128, 1500, 7, 30]],
                         ids=["2 behind 4000", "few before 20000", "mixed"])
def test_short_sequences_beside_long_ones(cuda_lib, lens, d, dtype):
    """The sequences of up to 128 tokens alone: dq and dk at most 1.3 times as far off the 64-bit result as the
    outputs' own rounding.

    A rounding's error has the same relative size e on average whatever is rounded, and e is what the output's
    has; ds rounded to the type would add a second independent one: sqrt(2) = 1.41 and more.  What stays
    is do.o from a P rounded once: with two tokens 0.71 e of dq at most, in all sqrt(1 + 0.5) = 1.22 (more
    tokens: smaller parts each); 6 % are for the sample."""
    leaves, cu, edges, dout = _inputs(lens, dtype, d, seed=len(lens) + d)
    grads = _grads(leaves, cu, dout)
    short = [(a, b) for a, b in zip(edges[:-1], edges[1:]) if b - a <= 128]
    rows = torch.cat([torch.arange(a, b, device="cuda") for a, b in short])
    own = [0]
    for a, b in short:
        own.append(own[-1] + b - a)
    ref = reference(*(t[rows] for t in leaves), own, -1, 0, 1 / math.sqrt(d), dout[rows])
    for name, got in (("dq", grads[0]), ("dk", grads[1])):
        want = ref[name][0]
        rounding = (want.to(dtype).double() - want).norm()
        assert float((got[rows].double() - want).norm() / rounding) <= 1.3, name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[200, 250], [90, 40, 3], [300, 290]], ids=str)
def test_rows_behind_the_last_sequence_change_no_bit(cuda_lib, monkeypatch, lens, dtype):
    """(The order of the sums over the group's heads goes by the token count: one share each.)"""
    monkeypatch.setenv("STEW_ATTN_SPLIT", "1")
    n = sum(lens)
    want = None
    for pad in (0, 1, 130, 2000):
        leaves, cu, _, dout = _inputs(lens, dtype, 128, pad)
        grads = _grads(leaves, cu, dout)
        assert not any(bool(g[n:].any()) for g in grads)
        grads = [g[:n] for g in grads]
        want = want or grads
        assert all(torch.equal(a, b) for a, b in zip(grads, want)), pad
