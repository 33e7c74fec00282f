"""CPU: the attention's backward launches with the addresses and strides of the tensors that autograd
hands back, which under checkpointing, offload and other saved-tensor hooks are not the forward's.
The launches are recorded instead of run."""
import ctypes

import pytest
import torch
from torch.utils.checkpoint import checkpoint


@pytest.fixture
def launches(monkeypatch):
    """[(entry, nf4b_attn, the other arguments)] of every launch, which does nothing."""
    from stew_b200 import _lib, step_ops
    seen = []

    def record(fn, what, device, rec, *args):
        seen.append((what, _lib.AttnC.from_buffer_copy(rec), args))

    monkeypatch.setattr(step_ops, "_launch", record)
    monkeypatch.setattr(step_ops, "packed_attention_supported", lambda q: True)
    return seen


def _inputs(fused):
    x = torch.zeros(24, 8, 64, dtype=torch.float16)
    q, k, v = x.split([4, 2, 2], dim=1)
    if not fused:
        q, k, v = q.clone(), k.clone(), v.clone()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    return leaves, torch.tensor([0, 10, 24], dtype=torch.int32)


def _fields(a, names):
    return tuple(getattr(a, n) for n in names.split())


SCALARS = "tokens rows heads kv_heads head_dim dtype left right scale"


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("odd", [False, True])
def test_backward_reads_the_unpacked_tensors(launches, fused, odd):
    """Hooks that move every saved tensor (odd: to an address that is not 16-byte aligned, so that it is
    copied once more): the backward names the unpacked ones, with their strides."""
    from stew_b200.step_ops import packed_attention
    leaves, cu = _inputs(fused)
    unpacked = []

    def unpack(t):
        if odd:
            buf = torch.empty(t.numel() + 1, dtype=t.dtype)
            buf[1:].view(t.shape).copy_(t)
            t = buf[1:].view(t.shape)
        unpacked.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().contiguous().clone(), unpack):
        out = packed_attention(*leaves, cu, window=(7, 3), scale=0.25)
    out.sum().backward()
    (w0, fwd, _), (w1, bwd, args) = launches
    assert (w0, w1) == ("nf4b_attn_fwd", "nf4b_attn_bwd")
    assert _fields(fwd, SCALARS) == _fields(bwd, SCALARS)
    assert _fields(bwd, "q_stride q_head_stride k_stride k_head_stride v_stride v_head_stride") == (256, 64, 128, 64, 128, 64)
    read = [bwd.q, bwd.k, bwd.v, bwd.cu, *args[:3]]  # and out, rest, lse
    if odd:
        assert all(a % 16 == 0 for a in read if a != bwd.cu)
        old = {fwd.q, fwd.k, fwd.v, fwd.cu}
        assert not old & set(read)
    else:
        assert set(read) == {t.data_ptr() for t in unpacked} and len(unpacked) == 7


@pytest.mark.parametrize("fused", [False, True])
def test_backward_under_checkpointing(launches, fused):
    """The recomputed forward's tensors are the ones that the backward reads."""
    from stew_b200.step_ops import packed_attention
    leaves, cu = _inputs(fused)
    alive = []

    def layer(q, k, v):
        kept = [t * 1.0 for t in (q, k, v)]
        alive.extend(kept)
        return packed_attention(*kept, cu)

    checkpoint(layer, *leaves, use_reentrant=False).sum().backward()
    names = [what for what, *_ in launches]
    assert names == ["nf4b_attn_fwd", "nf4b_attn_fwd", "nf4b_attn_bwd"]
    first, again, bwd = (a for _, a, _ in launches)
    assert _fields(bwd, "q k v cu") == _fields(again, "q k v cu")
    assert not set(_fields(first, "q k v")) & set(_fields(bwd, "q k v"))
    assert launches[2][2][0] == launches[1][2][0] and launches[2][2][2] == launches[1][2][2]  # out, lse


def test_plain_backward_reads_the_inputs(launches):
    """Without hooks nothing is copied: slices of one projection output are read in place."""
    from stew_b200.step_ops import packed_attention
    leaves, cu = _inputs(True)
    packed_attention(*leaves, cu).sum().backward()
    (_, fwd, _), (_, bwd, _) = launches
    assert bytes(fwd) == bytes(bwd)
    assert _fields(bwd, "q k v cu") == tuple(t.data_ptr() for t in (*leaves, cu))
    assert bwd.q_stride == 512 and ctypes.sizeof(bwd) == ctypes.sizeof(fwd)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_tangents_are_refused(launches, which, grad):
    """A dual tensor among q, k, v raises, with and without gradients: the result would carry no tangent."""
    import torch.autograd.forward_ad as fwad

    from stew_b200.step_ops import packed_attention
    leaves, cu = _inputs(False)
    qkv = [t.detach().requires_grad_(grad) for t in leaves]
    with fwad.dual_level():
        qkv[which] = fwad.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            packed_attention(*qkv, cu)
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
            packed_attention(*qkv, cu)
        packed_attention(*(t.detach() for t in leaves), cu)  # none of them dual: allowed


@pytest.mark.parametrize("scale", [3.5e38, 1e39, 1e300, 2.0 ** 127, 0.0, 1e-46, 5e-324, float("inf"), float("nan"), -1.0])
def test_scales_that_the_kernels_cannot_hold_are_refused(launches, scale):
    """The kernels take scale log2(e) in fp32."""
    from stew_b200.step_ops import packed_attention
    leaves, cu = _inputs(False)
    with pytest.raises(ValueError, match="scale"):
        packed_attention(*leaves, cu, scale=scale)
    assert not launches
    packed_attention(*leaves, cu, scale=1e38)
    assert len(launches) == 1


def test_scale_in_the_entry():
    from stew_b200 import _lib
    a = _lib.AttnC()
    a.q = a.k = a.v = a.cu = 256
    a.tokens, a.rows, a.heads, a.kv_heads, a.head_dim = 10, 1, 4, 2, 64
    a.q_stride, a.k_stride, a.v_stride = 256, 128, 128
    a.q_head_stride = a.k_head_stride = a.v_head_stride = 64
    a.dtype, a.left, a.right = _lib.NF4B_F16, -1, 0
    for scale, ok in ((1e38, True), (2.0 ** 127, False), (3.4e38, False)):
        a.scale = scale
        assert (_lib.lib().nf4b_attn_bwd_work_bytes(bytes(a)) > 0) == ok
