"""CPU: the argument checks of packed attention and of gradient clipping, in the C entries (before
anything touches a device) and in the Python entry points."""
import ctypes

import pytest
import torch


def _attn(**kw):
    from stew_b200 import _lib
    a = _lib.AttnC()
    a.q = a.k = a.v = a.cu = 256
    a.tokens, a.rows, a.heads, a.kv_heads, a.head_dim = 10, 1, 4, 2, 64
    a.q_stride, a.q_head_stride = 256, 64
    a.k_stride, a.k_head_stride = 128, 64
    a.v_stride, a.v_head_stride = 128, 64
    a.dtype, a.left, a.right, a.scale = _lib.NF4B_F16, -1, 0, 0.125
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(tokens=-1), "INVALID_ARG"), (dict(rows=-1), "INVALID_ARG"), (dict(heads=0), "INVALID_ARG"),
    (dict(kv_heads=3), "INVALID_ARG"), (dict(head_dim=0), "INVALID_ARG"), (dict(scale=0.0), "INVALID_ARG"),
    (dict(scale=-1.0), "INVALID_ARG"), (dict(scale=float("nan")), "INVALID_ARG"), (dict(scale=float("inf")), "INVALID_ARG"),
    (dict(q=None), "INVALID_ARG"), (dict(cu=None), "INVALID_ARG"),
    (dict(dtype=1), "UNSUPPORTED"), (dict(head_dim=60), "UNSUPPORTED"), (dict(head_dim=136), "UNSUPPORTED"),
    (dict(tokens=1 << 40), "UNSUPPORTED"), (dict(heads=1 << 20, kv_heads=1 << 20), "UNSUPPORTED"),
    (dict(k=264), "ALIGNMENT"), (dict(cu=258), "ALIGNMENT"), (dict(q_stride=260), "ALIGNMENT"),
    (dict(v_head_stride=0), "ALIGNMENT"), (dict(k_stride=-128), "ALIGNMENT"),
], ids=str)
def test_attention_entry_refuses(change, status):
    from stew_b200 import _lib
    L = _lib.lib()
    a, want = _attn(**change), getattr(_lib, "NF4B_ERR_" + status)
    assert L.nf4b_attn_fwd(ctypes.byref(a), 256, None, 256, None) == want
    assert L.nf4b_attn_bwd(ctypes.byref(a), 256, None, 256, 256, 256, 256, 256, 256, 1 << 30, None) == want


def test_attention_entry_refuses_buffers():
    from stew_b200 import _lib
    L = _lib.lib()
    a = ctypes.byref(_attn())
    assert L.nf4b_attn_fwd(None, 256, None, 256, None) == _lib.NF4B_ERR_INVALID_ARG
    assert L.nf4b_attn_fwd(a, None, None, 256, None) == _lib.NF4B_ERR_INVALID_ARG
    assert L.nf4b_attn_fwd(a, 264, None, 256, None) == _lib.NF4B_ERR_ALIGNMENT
    assert L.nf4b_attn_fwd(a, 256, 264, 256, None) == _lib.NF4B_ERR_ALIGNMENT
    need = L.nf4b_attn_bwd_work_bytes(a)
    assert need >= 10 * 4 * 8
    for bad in (dict(kv_heads=3), dict(tokens=-1), dict(head_dim=60), dict(k_stride=4)):
        assert L.nf4b_attn_bwd_work_bytes(ctypes.byref(_attn(**bad))) == -1
    assert L.nf4b_attn_bwd_work_bytes(None) == -1
    assert L.nf4b_attn_bwd(a, 256, None, 256, 256, 256, 256, 256, 256, need - 1, None) == _lib.NF4B_ERR_INVALID_ARG
    assert L.nf4b_attn_bwd(a, 256, None, 256, 256, 256, 256, 256, None, need, None) == _lib.NF4B_ERR_INVALID_ARG
    assert L.nf4b_attn_bwd(a, 256, None, 256, 256, 256, 264, 256, 256, need, None) == _lib.NF4B_ERR_ALIGNMENT
    none = ctypes.byref(_attn(tokens=0, q=None, k=None, v=None, cu=None))
    assert L.nf4b_attn_fwd(none, None, None, None, None) == _lib.NF4B_OK


def test_packed_attention_refuses():
    from stew_b200 import _lib
    from stew_b200.step_ops import packed_attention
    q, k = torch.zeros(8, 4, 64, dtype=torch.float16), torch.zeros(8, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(_lib.NF4Unsupported):  # CPU tensors: the kernels are the only implementation
        packed_attention(q, k, k, cu)
    for bad in ((q[0], k, k), (q, k, k.float()), (q, k[:7], k[:7]), (q, k, k[..., :32]), (q[:, :3], k, k)):
        with pytest.raises(ValueError):
            packed_attention(*bad, cu)


def test_clip_entry_refuses():
    from stew_b200 import _lib
    L = _lib.lib()
    one = (_lib.GradC * 1)()
    one[0].src, one[0].dst, one[0].numel, one[0].dtype = 256, 256, 10, _lib.NF4B_F32
    wb = L.nf4b_clip_grads_work_bytes(1)
    assert wb > 0 and L.nf4b_clip_grads_work_bytes(-1) == -1

    def call(g=one, n=1, max_norm=1.0, div=None, norm=256, work=256, bytes_=wb):
        return L.nf4b_clip_grads(g, n, max_norm, div, norm, work, bytes_, None)

    assert call(n=-1) == _lib.NF4B_ERR_INVALID_ARG
    assert call(max_norm=-0.5) == _lib.NF4B_ERR_INVALID_ARG
    assert call(max_norm=float("nan")) == _lib.NF4B_ERR_INVALID_ARG
    assert call(norm=None) == _lib.NF4B_ERR_INVALID_ARG
    assert call(work=None) == _lib.NF4B_ERR_INVALID_ARG
    assert call(g=None) == _lib.NF4B_ERR_INVALID_ARG
    assert call(bytes_=wb - 1) == _lib.NF4B_ERR_INVALID_ARG
    assert call(work=260) == _lib.NF4B_ERR_ALIGNMENT
    assert call(div=2) == _lib.NF4B_ERR_ALIGNMENT
    for field, value, status in (("src", None, _lib.NF4B_ERR_INVALID_ARG), ("numel", -1, _lib.NF4B_ERR_INVALID_ARG),
                                 ("dtype", 9, _lib.NF4B_ERR_UNSUPPORTED), ("src", 258, _lib.NF4B_ERR_ALIGNMENT),
                                 ("dst", 258, _lib.NF4B_ERR_ALIGNMENT)):
        bad = (_lib.GradC * 1)()
        ctypes.memmove(bad, one, ctypes.sizeof(one))
        setattr(bad[0], field, value)
        assert call(g=bad) == status, field


def test_clip_grads_refuses():
    from stew_b200 import _lib
    from stew_b200.dp import clip_grads
    with pytest.raises(ValueError):
        clip_grads([], 1.0)
    with pytest.raises(ValueError):
        clip_grads([torch.zeros(3)], -1.0)
    with pytest.raises(ValueError):
        clip_grads([torch.zeros(3)], float("nan"))
    with pytest.raises(ValueError):
        clip_grads([torch.zeros(3)], 1.0, out=[])
    with pytest.raises(_lib.NF4Unsupported):
        clip_grads([torch.zeros(3)], 1.0)


def test_grad_table_layout():
    """clip_grads fills nf4b_grad as four 64-bit words."""
    from stew_b200 import _lib
    assert ctypes.sizeof(_lib.GradC) == 32
    g = _lib.GradC.from_buffer_copy((ctypes.c_int64 * 4)(11, 12, 13, _lib.NF4B_BF16))
    assert (g.src, g.dst, g.numel, g.dtype) == (11, 12, 13, _lib.NF4B_BF16)
