"""GPU: attention over packed rows (nf4b_attn_fwd / nf4b_attn_bwd, step_ops.packed_attention) against
the definition in 64 bits (tests/attention_ref.py, with the elementwise bounds derived there)."""
import math

import pytest
import torch

from tests.attention_ref import assert_within, reference, row_mask

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """No pipeline wait of the kernels ran out of time in any test."""
    from stew_b200 import _lib
    yield
    if torch.cuda.is_available():
        assert _lib.attn_error_flag() == 0


def _edges(lens):
    e = [0]
    for x in lens:
        e.append(e[-1] + x)
    return e


def _inputs(lens, hq, hk, d, dtype, pad=0, seed=0, fused=False, dscale=0.02):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(lens) + hq + d)
    edges = _edges(lens)
    n = edges[-1] + pad
    x = torch.randn(n, hq + 2 * hk, d, device="cuda", generator=g).to(dtype)
    q, k, v = x.split([hq, hk, hk], dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    dout = (torch.randn(n, hq, d, device="cuda", generator=g) * dscale).to(dtype)
    return q, k, v, torch.tensor(edges, dtype=torch.int32, device="cuda"), edges, dout


def _check(q, k, v, cu, edges, dout, window=(-1, 0), scale=None):
    from stew_b200.step_ops import packed_attention
    leaves = [t.detach().clone().requires_grad_(True) if t.is_contiguous() else t.detach().requires_grad_(True)
              for t in (q, k, v)]
    out = packed_attention(*leaves, cu, window=window, scale=scale)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        assert torch.equal(packed_attention(q, k, v, cu, window=window, scale=scale), out)
    sc = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    ref = reference(q, k, v, edges, window[0], window[1], sc, dout)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert got.dtype == q.dtype and torch.isfinite(got).all(), name
        assert_within(got, *ref[name], name)
        assert not got[edges[-1]:].any(), f"{name}: rows behind the last sequence"


LENS = [[1], [2, 1, 3], [127], [128], [129], [255, 257], [64, 0, 65, 0], [300, 17, 512, 1, 90], [1000]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_lengths_causal(cuda_lib, lens, dtype):
    q, k, v, cu, edges, dout = _inputs(lens, 4, 2, 128, dtype, pad=3)
    _check(q, k, v, cu, edges, dout)


@pytest.mark.parametrize("hq,hk", [(12, 2), (1, 1), (5, 5), (7, 1), (16, 4)])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 80, 96, 120, 128])
def test_heads_and_head_sizes(cuda_lib, hq, hk, d):
    q, k, v, cu, edges, dout = _inputs([130, 47], hq, hk, d, torch.float16, seed=3)
    _check(q, k, v, cu, edges, dout)


@pytest.mark.parametrize("window", [(-1, -1), (0, 0), (0, -1), (5, 0), (64, 64), (127, 1), (128, 0), (200, 300), (1000, 0),
                                    (0, 7)])
@pytest.mark.parametrize("dtype,d", [(torch.float16, 128), (torch.bfloat16, 64)])
def test_windows(cuda_lib, window, dtype, d):
    q, k, v, cu, edges, dout = _inputs([390, 128, 1, 33], 4, 1, d, dtype, seed=5)
    _check(q, k, v, cu, edges, dout, window=window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [8, 64, 72, 128])
@pytest.mark.parametrize("lens,window", [([390, 128, 1, 633], (-1, -1)), ([390, 128, 1, 633], (5, -1)), ([257], (64, 64)),
                                         ([700, 0, 333], (200, 300)), ([513, 512], (-1, 7)), ([260, 259], (-1, 0))], ids=str)
def test_longer_rows(cuda_lib, lens, window, d, dtype):
    """Sequences of more than 256 tokens on average (their ds is rounded once), with every kind of window."""
    q, k, v, cu, edges, dout = _inputs(lens, 6, 2, d, dtype, seed=7)
    assert edges[-1] > 256 * len(lens)
    _check(q, k, v, cu, edges, dout, window=window)


@pytest.mark.parametrize("split", ["1", "2", "3", "6"])
def test_shares_of_a_group_in_longer_rows(cuda_lib, monkeypatch, split):
    monkeypatch.setenv("STEW_ATTN_SPLIT", split)
    q, k, v, cu, edges, dout = _inputs([300, 517], 12, 2, 96, torch.float16, seed=8, pad=5)
    _check(q, k, v, cu, edges, dout)


@pytest.mark.parametrize("pad", [0, 1, 200])
def test_strided_projection_output_and_padding(cuda_lib, pad):
    q, k, v, cu, edges, dout = _inputs([77, 260], 6, 2, 64, torch.bfloat16, pad=pad, fused=True)
    assert not q.is_contiguous()
    _check(q, k, v, cu, edges, dout, window=(-1, -1))


def test_other_layouts_and_broadcast_heads(cuda_lib):
    """Head-major storage, an unaligned view and a key/value head broadcast over all heads give
    what their contiguous copies give; the broadcast input's gradient is the sum over the heads."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([150, 33], 4, 4, 64, torch.float16)
    want = packed_attention(q, k, v, cu)
    hm = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (q, k, v)]
    assert torch.equal(packed_attention(*hm, cu), want)
    buf = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
    odd = buf[1:].view_as(q)
    odd.copy_(q)
    assert odd.data_ptr() % 16 != 0
    assert torch.equal(packed_attention(odd, k, v, cu), want)
    wide = torch.randn(q.shape[0], 4, 130, device="cuda").half()  # token stride not a multiple of 8
    wide[..., :64] = q
    assert torch.equal(packed_attention(wide[..., :64], k, v, cu), want)
    one = k[:, :1].clone().requires_grad_(True)
    both = packed_attention(q, one.expand(-1, 4, -1), v, cu)
    (g,) = torch.autograd.grad(both, one, dout)
    full = k[:, :1].expand(-1, 4, -1).contiguous().requires_grad_(True)
    assert torch.equal(packed_attention(q, full, v, cu), both)
    (gf,) = torch.autograd.grad(packed_attention(q, full, v, cu), full, dout)
    assert torch.equal(g, gf.sum(1, keepdim=True))


@pytest.mark.parametrize("dscale", [1e-6, 1.0, 300.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradient_scales(cuda_lib, dscale, dtype):
    """Tiny and large gradients keep their precision: ds is scaled into fp16's range before its
    rounding.  The relative bound of the formulas holds where the outputs are normal numbers of
    the type; fp16's 2^-25 is in the bound."""
    q, k, v, cu, edges, dout = _inputs([200, 310], 4, 2, 128, dtype, dscale=dscale)
    _check(q, k, v, cu, edges, dout)


@pytest.mark.parametrize("window", [(64, 0), (0, 64)])
def test_gradient_scales_under_a_window(cuda_lib, window):
    """Rows whose gradients are 2^24 times smaller than those of a far part of their sequence, whose
    tiles no window joins to theirs, keep their precision: scaled by the far rows' size, a ds of
    about 2^-15 would be rounded to steps of 2^-20, where its bound here is 2^-26.

    Where a window does join tiles, all ds of a 128-token tile share one scale 2^k, with
    k = 14 - floor(log2 M) >= 14 - log2 M, M the largest |dO||V| + |delta| of the tiles that meet;
    a scaled ds below fp16's normal range is off by up to 2^-25, so ds by 2^-25 / 2^k <= M 2^-39,
    which the bounds of assert_within's reference (ds in the normal range) do not hold."""
    from stew_b200.step_ops import packed_attention
    n, hq, hk, d = 640, 4, 2, 64
    q, k, v, cu, edges, dout = _inputs([n], hq, hk, d, torch.float16, seed=21, dscale=2.0 ** -12)
    dout[:128] *= 2.0 ** 24
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, cu, window=window)
    grads = torch.autograd.grad(out, leaves, dout)
    sc = 1 / math.sqrt(d)
    ref = reference(q, k, v, edges, *window, sc, dout)
    see = row_mask(n, *window, "cuda").double()
    tiles = n // 128
    n_do, n_v = dout.double().norm(dim=2), v.double().norm(dim=2)  # [n, hq], [n, hk]
    delta = (dout.double() * ref["out"][0]).sum(2).abs()
    size = lambda x, t, m: x[t * 128:(t + m) * 128].amax(0)  # of tiles [t, t + m), by head
    for t in range(tiles):
        mine = slice(t * 128, (t + 1) * 128)
        for keys in (False, True):
            back, ahead = window[::-1] if keys else window
            lo, hi = max(0, t * 128 - back) // 128, min(n - 1, t * 128 + 127 + ahead) // 128
            a, b = ((lo, hi - lo + 1), (t, 1)) if keys else ((t, 1), (lo, hi - lo + 1))
            m = size(n_do, *a) * size(n_v, *b).repeat_interleave(hq // hk) + size(delta, *a)  # [hq]
            lost = sc * m * 2.0 ** -39
            if keys:  # over the group's heads, one scale for all of them at most
                lost = lost.view(hk, -1).amax(1)[:, None]
                x = q.double().abs().view(n, hk, hq // hk, d).sum(2)
                ref["dk"][1][mine] += lost * torch.einsum("ij,ihd->jhd", see[:, mine], x)
            else:
                x = k.double().abs().repeat_interleave(hq // hk, 1)
                ref["dq"][1][mine] += lost[:, None] * torch.einsum("ij,jhd->ihd", see[mine], x)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,window,d", [([2] * 40, (-1, 0), 128), ([1, 3, 5, 2, 70, 128, 0, 9], (-1, 0), 64),
                                           ([128, 100], (-1, -1), 96), ([500, 131], (2, 0), 128), ([700], (60, 67), 64),
                                           ([300] + [1] * 9, (-1, 0), 128)], ids=str)
def test_few_tokens_keep_what_the_rounding_of_ds_leaves(cuda_lib, lens, window, d, dtype):
    """Where the tokens see few others on average, dq and dk are as if ds were not rounded to the type:
    1.3 times as far off as the output's own rounding at most, over all elements.

    A rounding's error has the same relative size e on average, whatever is rounded, and e is what the
    output's has.  ds rounded to the type would add a second independent e: sqrt(2) = 1.41 and more.
    What stays is do.o: o = (V_m + sum_j r(p_j) V_j) / l holds the roundings of all p but the
    largest (exp(0) = 1).  With two tokens, p_2 <= p_1, dO of size s and d features, that shifts do.o by
    e p_2 s sqrt(d) and so dq by e p_2 s sqrt(d) sqrt(p_1^2 + p_2^2) |K|, against dq =
    p_1 p_2 (dP_1 - dP_2) (K_1 - K_2) of size 2 p_1 p_2 s sqrt(d) |K|: e sqrt(p_1^2 + p_2^2) / (2 p_1)
    <= 0.71 e, in all sqrt(1 + 0.5) = 1.22 (more tokens: smaller parts each); 6 % are for the sample."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs(lens, 4, 2, d, dtype, seed=31)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, cu, window=window)
    grads = torch.autograd.grad(out, leaves, dout)
    ref = reference(q, k, v, edges, *window, 1 / math.sqrt(d), dout)
    for name, got in (("dq", grads[0]), ("dk", grads[1])):
        want = ref[name][0]
        own = (want.to(dtype).double() - want).norm()
        assert float((got.double() - want).norm() / own) <= 1.3, name


def test_large_scores_and_values(cuda_lib):
    """Scores up to some hundreds (one-hot rows), large values."""
    q, k, v, cu, edges, dout = _inputs([257, 140], 4, 2, 128, torch.float16, seed=9)
    _check(q * 6, k * 6, v * 100, cu, edges, dout, scale=1 / math.sqrt(128) / 4)
    _check(q, k, v, cu, edges, dout, scale=1e-4)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 65504.0])
def test_other_rows_values_stay_out(cuda_lib, bad):
    """A sequence is not touched by what its neighbours in the packed buffer, or the rows behind
    the last one, hold: NaN and infinities there leave its output and gradients bit for bit."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([70, 61, 200], 4, 2, 128, torch.float16, pad=9)
    a, b = edges[1], edges[2]

    def run(q, k, v, dout):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        o = packed_attention(*leaves, cu)
        return (o.detach(), *torch.autograd.grad(o, leaves, dout))

    want = run(q, k, v, dout)
    others = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    others[a:b] = False
    got = run(*(torch.where(others[:, None, None], torch.full_like(t, bad), t) for t in (q, k, v, dout)))
    for w, g in zip(want, got):
        assert torch.equal(w[a:b], g[a:b])
        assert not g[edges[-1]:].any()


def test_masked_keys_inside_a_sequence(cuda_lib):
    """A NaN key or query that the window hides from a token does not reach it."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, _ = _inputs([300], 2, 1, 128, torch.float16)
    want = packed_attention(q, k, v, cu)
    k2 = k.clone()
    k2[200:] = float("nan")
    got = packed_attention(q, k2, v, cu)
    assert torch.equal(got[:200], want[:200]) and torch.isnan(got[200:]).all()


def test_same_bits_on_every_run(cuda_lib):
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([900, 301, 700], 12, 2, 128, torch.float16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def run():
        o = packed_attention(*leaves, cu)
        return (o.detach(), *torch.autograd.grad(o, leaves, dout))

    first = run()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_differences(cuda_lib):
    """The gradient against central differences of the 64-bit definition's loss along random
    directions: the directional derivative within the gradient's own error bound."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([90, 41], 4, 2, 64, torch.float16, seed=11, dscale=1.0)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, cu), leaves, dout)
    ref = reference(q, k, v, edges, -1, 0, 1 / 8, dout)
    x = [t.double() for t in (q, k, v)]
    g = torch.Generator(device="cuda").manual_seed(4)
    step = 1e-5
    for i, name in enumerate(("dq", "dk", "dv")):
        u = torch.randn(x[i].shape, generator=g, device="cuda", dtype=torch.float64)
        loss = []
        for s in (step, -step):
            y = list(x)
            y[i] = x[i] + s * u
            loss.append(float((reference64(*y, edges) * dout.double()).sum()))
        slope = (loss[0] - loss[1]) / (2 * step)
        bound = float((1.05 * ref[name][1] * u.abs()).sum()) + 1e-6 * abs(slope) + 1e-6
        assert abs(float((grads[i].double() * u).sum()) - slope) <= bound, name


def reference64(q, k, v, edges):
    out = torch.zeros_like(q)
    grp = q.shape[1] // k.shape[1]
    for a, b in zip(edges[:-1], edges[1:]):
        see = torch.tril(torch.ones(b - a, b - a, dtype=torch.bool, device=q.device))
        for h in range(q.shape[1]):
            s = (q[a:b, h] @ k[a:b, h // grp].T / 8).masked_fill(~see, float("-inf"))
            out[a:b, h] = torch.softmax(s, -1) @ v[a:b, h // grp]
    return out


def test_many_sequences_and_no_sequence(cuda_lib):
    from stew_b200.step_ops import packed_attention
    lens = [(i * 7) % 5 for i in range(700)]
    q, k, v, cu, edges, dout = _inputs(lens, 2, 1, 64, torch.bfloat16)
    _check(q, k, v, cu, edges, dout)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not packed_attention(q, k, v, none).any()
    empty = [t[:0].requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*empty, none)
    assert out.shape == (0, 2, 64)
    assert [g.shape for g in torch.autograd.grad(out.sum(), empty)] == [(0, 2, 64), (0, 1, 64), (0, 1, 64)]


def test_row_starts_out_of_range_are_cut(cuda_lib):
    """Starts past the buffer or below zero address nothing outside it."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([100, 60], 2, 1, 64, torch.float16)
    want = packed_attention(q, k, v, cu)
    far = torch.tensor([0, 100, 2_000_000_000], dtype=torch.int32, device="cuda")
    assert torch.equal(packed_attention(q, k, v, far), want)
    neg = torch.tensor([0, -5, 160], dtype=torch.int32, device="cuda")
    whole = packed_attention(q, k, v, torch.tensor([0, 160], dtype=torch.int32, device="cuda"))
    assert torch.equal(packed_attention(q, k, v, neg), whole)


def test_captured_and_replayed_on_a_side_stream(cuda_lib):
    """Forward and backward captured into a graph while an eager graph of the same leaves lives;
    the replay on new inputs gives the eager result, bit for bit."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([250, 131], 4, 2, 128, torch.float16)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    alive = packed_attention(*leaves, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        static = [t.detach().clone().requires_grad_(True) for t in leaves]
        o = packed_attention(*static, cu)
        torch.autograd.grad(o, static, dout)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = packed_attention(*static, cu)
        grads = torch.autograd.grad(o, static, dout)
    q2, k2, v2, *_ = _inputs([250, 131], 4, 2, 128, torch.float16, seed=77)
    with torch.no_grad():
        for s, t in zip(static, (q2, k2, v2)):
            s.copy_(t)
    g.replay()
    eager = [t.clone().requires_grad_(True) for t in (q2, k2, v2)]
    oe = packed_attention(*eager, cu)
    ge = torch.autograd.grad(oe, eager, dout)
    assert torch.equal(o, oe) and all(torch.equal(a, b) for a, b in zip(grads, ge))
    assert torch.isfinite(torch.autograd.grad(alive, leaves, dout)[0]).all()


def test_two_streams_at_once(cuda_lib):
    from stew_b200.step_ops import packed_attention
    sets = [_inputs([600, 200], 4, 2, 128, torch.float16, seed=s) for s in (1, 2)]
    want = [packed_attention(*s[:4]) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(packed_attention(*s[:4]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for w, os in zip(want, got) for o in os)


def test_two_backwards_at_once(cuda_lib, monkeypatch):
    """Backward passes whose CTAs wait for sums over shares, on three streams at once: neither holds
    the other up."""
    from stew_b200 import _lib
    from stew_b200.step_ops import packed_attention
    monkeypatch.setenv("STEW_ATTN_SPLIT", "6")
    sets = [_inputs([900, 400, 700], 12, 2, 128, torch.float16, seed=s) for s in (1, 2, 3)]

    def run(s):
        leaves = [t.detach().requires_grad_(True) for t in s[:3]]
        return torch.autograd.grad(packed_attention(*leaves, s[3]), leaves, s[5])

    want = [run(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]
    for _ in range(6):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(run(s))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(a, b) for g in gs for a, b in zip(w, g))
    assert _lib.attn_error_flag() == 0


@pytest.mark.parametrize("split", ["1", "2", "3", "6"])
@pytest.mark.parametrize("d", [64, 80, 128])
def test_shares_of_a_group(cuda_lib, monkeypatch, split, d):
    """A key tile's heads on one CTA or shared out over several."""
    monkeypatch.setenv("STEW_ATTN_SPLIT", split)
    q, k, v, cu, edges, dout = _inputs([300, 140, 1, 129], 6, 1, d, torch.float16, pad=5, seed=8)
    _check(q, k, v, cu, edges, dout)


def test_one_token_dimension_with_any_stride(cuda_lib):
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([1], 1, 1, 64, torch.float16)
    want = packed_attention(q, k, v, cu)
    odd = [t.as_strided((1, 1, 64), (3, 5, 1)) for t in (q, k, v)]
    assert torch.equal(packed_attention(*odd, cu), want) and torch.equal(want, v)


def test_changed_row_starts_are_noticed(cuda_lib):
    """The row starts are saved for the backward; changing them in between is an error, not a wrong
    gradient."""
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([20, 30], 1, 1, 64, torch.float16)
    q.requires_grad_(True)
    out = packed_attention(q, k, v, cu)
    cu[1] = 10
    with pytest.raises(RuntimeError):
        out.backward(dout)


def test_long_row_past_32_bit_offsets(cuda_lib):
    """q's rows lie more than 2^31 elements apart from its base: a token stride of 2^18 elements
    over 9,000 tokens.  A narrow window keeps the reference small."""
    from stew_b200.step_ops import packed_attention
    n, d = 9000, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    big = torch.empty(n, 1 << 18, dtype=torch.float16, device="cuda")
    q = big[:, :d].view(n, 1, d)
    q.copy_(torch.randn(n, 1, d, device="cuda", generator=g))
    k, v = (torch.randn(n, 1, d, device="cuda", generator=g).half() for _ in range(2))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = packed_attention(q, k, v, cu, window=(3, 0))
    assert torch.equal(got, packed_attention(q.contiguous(), k, v, cu, window=(3, 0)))
    tail = reference(q[-200:], k[-200:], v[-200:], [0, 200], 3, 0, 1 / 8)["out"]
    assert_within(got[-100:], tail[0][100:], tail[1][100:], "out")


def test_no_second_derivative(cuda_lib):
    from stew_b200.step_ops import packed_attention
    q, k, v, cu, edges, dout = _inputs([20], 1, 1, 64, torch.float16)
    q.requires_grad_(True)
    (g,) = torch.autograd.grad(packed_attention(q, k, v, cu), q, dout, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().square().sum(), q)


def test_attention_of_the_step_after_rope(cuda_lib):
    """A run of the layer's operators as the step uses them: rotary embedding, attention, backward
    through both, against the 64-bit definition on the rotated tensors."""
    from stew_b200.qlora_step import rope_tables
    from stew_b200.step_ops import packed_attention, rope_qk
    q, k, v, cu, edges, dout = _inputs([180, 75], 12, 2, 128, torch.float16)
    pos = torch.cat([torch.arange(180), torch.arange(75)]).cuda()
    cos, sin = rope_tables(pos, 128, 1e6)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    qr, kr = rope_qk(q, k, cos, sin)
    out = packed_attention(qr, kr, v, cu)
    gq, gk, gv = torch.autograd.grad(out, leaves, dout)
    ref = reference(qr.detach(), kr.detach(), v.detach(), edges, -1, 0, 1 / math.sqrt(128), dout)
    assert_within(out.detach(), *ref["out"], "out")
    assert_within(gv, *ref["dv"], "dv")

    def unrotate(x):  # the rotation's transpose, and its absolute form for the bound
        c, s = cos.double()[:, None], sin.double()[:, None]
        a, b = x[..., :64], x[..., 64:]
        return torch.cat([a * c[..., :64] + b * s[..., 64:], b * c[..., 64:] - a * s[..., :64]], -1)

    def spread(x):
        a, b = x[..., :64], x[..., 64:]
        return torch.cat([a + b, a + b], -1)

    for got, name in ((gq, "dq"), (gk, "dk")):
        val, bound = ref[name]
        want = unrotate(val)
        assert_within(got, want, spread(bound) + 2.0 ** -11 * want.abs() + 2.0 ** -25, name)
