"""GPU: packed attention inside autograd's other machinery -- checkpointing, tensors saved on the CPU,
hooks that move what was saved: the gradients are those of a plain call, bit for bit (both run the
same kernels on the same values)."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

LENS = [130, 1, 0, 300, 77]


def _inputs(fused, dtype=torch.float16, seed=0, pad=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(LENS) + pad
    x = torch.randn(n, 8, 128, device="cuda", generator=g).to(dtype)
    q, k, v = x.split([4, 2, 2], dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cu = torch.tensor([0] + LENS, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
    return [t.detach().requires_grad_(True) for t in (q, k, v)], cu, torch.randn(n, 4, 128, device="cuda", generator=g).to(dtype)


def _churn():
    """Overwrites what the caching allocator has free: freed memory that is read shows."""
    kept = [torch.full((1 << s,), float("nan"), device="cuda") for s in range(8, 22) for _ in range(4)]
    del kept


def _plain(leaves, cu, dout, window):
    from stew_b200.step_ops import packed_attention
    return torch.autograd.grad(packed_attention(*leaves, cu, window=window), leaves, dout)


def _moved(t):
    """The same values elsewhere, in a layout of its own."""
    return t.detach().contiguous().clone()


def _misaligned(t):
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    buf[1:].view(t.shape).copy_(t)
    return buf[1:].view(t.shape)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window", [(-1, 0), (40, 9)])
@pytest.mark.parametrize("how", ["checkpoint", "cpu", "clone", "misaligned"])
def test_gradients_are_those_of_a_plain_call(cuda_lib, how, window, dtype, fused):
    from stew_b200.step_ops import packed_attention
    leaves, cu, dout = _inputs(fused, dtype)
    want = _plain(leaves, cu, dout, window)

    def layer(q, k, v):  # the attention reads tensors that only this call's graph holds
        return packed_attention(q * 1, k * 1, v * 1, cu.clone(), window=window)

    if how == "checkpoint":
        out = checkpoint(layer, *leaves, use_reentrant=False)
    elif how == "cpu":
        with torch.autograd.graph.save_on_cpu():
            out = layer(*leaves)
    else:
        with torch.autograd.graph.saved_tensors_hooks(_moved, _moved if how == "clone" else _misaligned):
            out = layer(*leaves)
    _churn()
    got = torch.autograd.grad(out, leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offloaded_slices_come_back_with_other_strides(cuda_lib):
    """The attention saves slices of one projection output; the hooks hand back contiguous tensors."""
    from stew_b200.step_ops import packed_attention
    leaves, cu, dout = _inputs(True)
    want = _plain(leaves, cu, dout, (-1, 0))
    with torch.autograd.graph.saved_tensors_hooks(_moved, _moved):
        out = packed_attention(*leaves, cu)
    _churn()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, dout), want))


def test_checkpointed_twice_in_a_row(cuda_lib):
    """Two layers of attention, each checkpointed: every recomputation uses its own tensors."""
    from stew_b200.step_ops import packed_attention
    leaves, cu, dout = _inputs(False)
    q, k, v = leaves

    def layer(x):
        return packed_attention(x, k, v, cu)

    want = torch.autograd.grad(layer(layer(q)), leaves, dout)
    out = checkpoint(layer, checkpoint(layer, q, use_reentrant=False), use_reentrant=False)
    _churn()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, dout), want))
