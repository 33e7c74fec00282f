"""Autograd wrappers of the layer kernels of the packed-token QLoRA step (C ABI
include/stew_step.h): RMSNorm, RMSNorm fused with the residual add, rotary embedding of q and
k, attention over packed rows, SwiGLU and the LM head's cross-entropy -- the counterparts of the
reference's
solution/rmsnorm.py (RMSNormFn :59-92, AddRMSNormFn :192-233), solution/rope.py (:71-92),
solution/swiglu.py (:42-66) and solution/head_loss.py.  fp16 activations, fp32 math; the CUDA
kernels are the only implementation (no torch fallback)."""
from __future__ import annotations

import ctypes
import math
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .nf4 import _launch, _stream


def _c(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _w32(w: torch.Tensor) -> torch.Tensor:
    return _c(w if w.dtype == torch.float32 else w.float())


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        x2 = _c(x.reshape(-1, x.shape[-1]))
        w32 = _w32(w)
        rows, hidden = x2.shape
        y = torch.empty_like(x2)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        _lib.check(_lib.lib().nf4b_rmsnorm_fwd(x2.data_ptr(), None, w32.data_ptr(), float(eps), None,
                                               y.data_ptr(), rstd.data_ptr(), rows, hidden,
                                               _stream(x.device)), "nf4b_rmsnorm_fwd")
        ctx.save_for_backward(x2, w32, rstd)
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w32, rstd = ctx.saved_tensors
        rows, hidden = x2.shape
        dy2 = _c(dy.reshape(rows, hidden).to(torch.float16))
        dx = torch.empty_like(x2)
        _lib.check(_lib.lib().nf4b_rmsnorm_bwd(dy2.data_ptr(), x2.data_ptr(), w32.data_ptr(),
                                               rstd.data_ptr(), None, dx.data_ptr(), rows, hidden,
                                               _stream(dx.device)), "nf4b_rmsnorm_bwd")
        return dx.view(ctx.shape), None, None


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, res, delta, w, eps):
        r2 = _c(res.reshape(-1, res.shape[-1]))
        d2 = _c(delta.reshape(r2.shape))
        w32 = _w32(w)
        rows, hidden = r2.shape
        s = torch.empty_like(r2)
        y = torch.empty_like(r2)
        rstd = torch.empty(rows, dtype=torch.float32, device=res.device)
        _lib.check(_lib.lib().nf4b_rmsnorm_fwd(r2.data_ptr(), d2.data_ptr(), w32.data_ptr(), float(eps),
                                               s.data_ptr(), y.data_ptr(), rstd.data_ptr(), rows,
                                               hidden, _stream(res.device)), "nf4b_rmsnorm_fwd")
        ctx.save_for_backward(s, w32, rstd)
        ctx.shape = res.shape
        return s.view(res.shape), y.view(res.shape)

    @staticmethod
    def backward(ctx, ds, dy):
        s, w32, rstd = ctx.saved_tensors
        rows, hidden = s.shape
        dx = torch.empty_like(s)
        if dy is None:  # only the residual stream is used downstream
            dx.copy_(ds.reshape(rows, hidden))
        else:
            dy2 = _c(dy.reshape(rows, hidden).to(torch.float16))
            ds2 = None if ds is None else _c(ds.reshape(rows, hidden).to(torch.float16))
            _lib.check(_lib.lib().nf4b_rmsnorm_bwd(dy2.data_ptr(), s.data_ptr(), w32.data_ptr(),
                                                   rstd.data_ptr(), None if ds2 is None else ds2.data_ptr(),
                                                   dx.data_ptr(), rows, hidden, _stream(dx.device)),
                       "nf4b_rmsnorm_bwd")
        dxv = dx.view(ctx.shape)
        return dxv, dxv, None, None


class _RopeQK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin):
        q, k = _c(q), _c(k)
        cos32, sin32 = _c(cos.float()), _c(sin.float())
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        _RopeQK._run(q, k, cos32, sin32, qo, ko, 0)
        ctx.save_for_backward(cos32, sin32)
        return qo, ko

    @staticmethod
    def _run(q, k, cos32, sin32, qo, ko, inverse):
        t, hq, d = q.shape
        _lib.check(_lib.lib().nf4b_rope_qk(q.data_ptr(), k.data_ptr(), cos32.data_ptr(), sin32.data_ptr(),
                                           qo.data_ptr(), ko.data_ptr(), t, hq, k.shape[1], d, inverse,
                                           _stream(q.device)), "nf4b_rope_qk")

    @staticmethod
    def backward(ctx, dq, dk):
        cos32, sin32 = ctx.saved_tensors
        dq = _c(dq.to(torch.float16))
        dk = _c(dk.to(torch.float16))
        gq, gk = torch.empty_like(dq), torch.empty_like(dk)
        _RopeQK._run(dq, dk, cos32, sin32, gq, gk, 1)
        return gq, gk, None, None


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        g, u = _c(gate), _c(up)
        m = torch.empty_like(g)
        _lib.check(_lib.lib().nf4b_swiglu_fwd(g.data_ptr(), u.data_ptr(), m.data_ptr(), g.numel(),
                                              _stream(g.device)), "nf4b_swiglu_fwd")
        ctx.save_for_backward(g, u)
        return m

    @staticmethod
    def backward(ctx, dm):
        g, u = ctx.saved_tensors
        dm = _c(dm.to(torch.float16))
        dg, du = torch.empty_like(g), torch.empty_like(u)
        _lib.check(_lib.lib().nf4b_swiglu_bwd(dm.data_ptr(), g.data_ptr(), u.data_ptr(), dg.data_ptr(),
                                              du.data_ptr(), g.numel(), _stream(g.device)),
                   "nf4b_swiglu_bwd")
        return dg, du


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """fp16(w * fp16(x * rsqrt(mean(x^2) + eps))) over the last dimension."""
    return _RMSNorm.apply(x, w, eps)


def add_rms_norm(res: torch.Tensor, delta: torch.Tensor, w: torch.Tensor, eps: float):
    """(s, rms_norm(s)) with s = fp16(res + delta): the residual add and the next norm."""
    return _AddRMSNorm.apply(res, delta, w, eps)


def rope_qk(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
    """Rotary embedding (rotate-half) of q [T, Hq, D] and k [T, Hk, D]; cos/sin [T, D]."""
    return _RopeQK.apply(q, k, cos, sin)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """fp16(gate * sigmoid(gate) * up), fp32 inside (the reference's SwiGLU kernel)."""
    return _SwiGLU.apply(gate, up)


ATTN_MAX_HEAD_DIM = 128
_ATTN_DTYPE = {torch.float16: _lib.NF4B_F16, torch.bfloat16: _lib.NF4B_BF16}


def _aligned_c(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _attn_layout(t: torch.Tensor) -> tuple:
    """(t, token stride, head stride) of t [tokens, heads, head_dim] as the kernels read it:
    contiguous features, strides that are multiples of 8 elements, a 16-byte aligned base (slices
    of one projection output stay as they are; anything else, a broadcast view too, is copied)."""
    n, h, d = t.shape
    st, sh, sd = t.stride()
    # a dimension of one element may carry any stride
    st, sh = (st if n > 1 else h * d), (sh if h > 1 else d)
    if sd == 1 and st >= d and sh >= d and not (st | sh) & 7 and not t.data_ptr() & 15:
        return t, st, sh
    return _aligned_c(t), h * d, d


# nf4b_attn as one packed record (a quarter of the time of filling a ctypes structure)
_ATTN_RECORD = struct.Struct("=4Q7q7if")
assert _ATTN_RECORD.size == ctypes.sizeof(_lib.AttnC)


def _attn_record(q, qs, k, ks, v, vs, cu, left, right, scale) -> bytes:
    n, hq, d = q.shape
    return _ATTN_RECORD.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu.data_ptr(), n, *qs, *ks, *vs,
                             cu.numel() - 1, hq, k.shape[1], d, _ATTN_DTYPE[q.dtype], left, right, scale)


def _attn_forward(q, k, v, cu, left, right, scale, keep_rest=False):
    """(out, what its rounding left or None, lse, q, k, v as read)."""
    q, *qs = _attn_layout(q)
    k, *ks = _attn_layout(k)
    v, *vs = _attn_layout(v)
    n, hq, _ = q.shape
    dev = q.device
    # (empty_like with a memory format is less than half the host time of empty with a Size)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    rest = torch.empty_like(q, memory_format=torch.contiguous_format) if keep_rest else None
    lse = torch.empty(hq, n, dtype=torch.float32, device=dev)
    if n:
        rec = _attn_record(q, qs, k, ks, v, vs, cu, left, right, scale)
        _launch(_lib.lib().nf4b_attn_fwd, "nf4b_attn_fwd", dev, rec, out.data_ptr(),
                rest.data_ptr() if keep_rest else None, lse.data_ptr())
    return out, rest, lse, q, k, v


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, left, right, scale):
        out, rest, lse, q, k, v = _attn_forward(q, k, v, cu, left, right, scale, True)
        ctx.save_for_backward(q, k, v, cu, out, rest, lse)
        ctx.scalars = left, right, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        # Under checkpointing, offload and other saved-tensor hooks these are not the tensors that the
        # forward read: their addresses and strides are taken here, and nothing of the forward's.
        q, k, v, cu, out, rest, lse = ctx.saved_tensors
        dev, dt = q.device, q.dtype
        q, *qs = _attn_layout(q)
        k, *ks = _attn_layout(k)
        v, *vs = _attn_layout(v)
        cu = cu.contiguous()
        out, rest, lse = _aligned_c(out), _aligned_c(rest), _aligned_c(lse)
        dout = _aligned_c(dout if dout.dtype == dt else dout.to(dt))
        dq = torch.empty_like(q, memory_format=torch.contiguous_format)
        dk = torch.empty_like(k, memory_format=torch.contiguous_format)
        dv = torch.empty_like(v, memory_format=torch.contiguous_format)
        if q.shape[0]:
            L = _lib.lib()
            rec = _attn_record(q, qs, k, ks, v, vs, cu, *ctx.scalars)
            wb = L.nf4b_attn_bwd_work_bytes(rec)
            work = torch.empty(wb, dtype=torch.uint8, device=dev)
            _launch(L.nf4b_attn_bwd, "nf4b_attn_bwd", dev, rec, out.data_ptr(), rest.data_ptr(), lse.data_ptr(),
                    dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), work.data_ptr(), wb)
        return dq, dk, dv, None, None, None, None


def _dual_level() -> bool:
    """Whether a forward-mode level is open (1 us less than asking three tensors)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def packed_attention_supported(q: torch.Tensor) -> bool:
    """Whether packed_attention's kernels take q's type and head size."""
    return (q.is_cuda and q.dtype in _ATTN_DTYPE and q.shape[-1] % 8 == 0
            and 0 < q.shape[-1] <= ATTN_MAX_HEAD_DIM)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, window=(-1, 0),
                     scale: float | None = None) -> torch.Tensor:
    """Attention inside each of the sequences packed one after the other in q [N, Hq, D] and
    k, v [N, Hk, D] (fp16 or bf16; D a multiple of 8 up to 128; Hq a multiple of Hk, query head h
    reading key/value head h // (Hq / Hk)).  cu: int32 [B + 1] on the same device, sequence b is
    tokens [cu[b], cu[b+1]), cu[0] = 0, ascending; empty sequences are allowed.  Its values are
    not read on the host: the kernels cut them to [0, N].
    window = (left, right): token i sees the tokens i - left <= j <= i + right of its sequence, -1
    for no bound; (-1, 0) is causal, (-1, -1) sees everything.  scale: of the scores, default
    1 / sqrt(D).
    Returns [N, Hq, D]; tokens behind cu[B] get zeros, and zero gradients.  What other sequences hold,
    NaN too, does not reach a token; a NaN or infinity in v or in the output's gradient may reach
    tokens of its own sequence that do not see it.  Any strides with contiguous features are read in
    place when they are multiples of 8 elements, else copied.
    The backward recomputes the probabilities from the saved log-sum-exp; beside the output it
    keeps what the output's rounding left (a second tensor of its size), so that the rows' do.o
    are free of it.  Forward and backward give the same bits on every run (the order of the fp32
    sums goes by the counts of tokens, sequences and heads).  Second derivatives and forward-mode
    tangents are refused.  A wait inside a kernel that runs out of time leaves NaN in the rows
    concerned; _lib.raise_if_wait_ran_out() tells."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("packed_attention: q, k and v must be [tokens, heads, head_dim]")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        raise ValueError("packed_attention: q, k and v must share one type and device")
    n, hq, d = q.shape
    if k.shape != v.shape or k.shape[0] != n or k.shape[2] != d:
        raise ValueError(f"packed_attention: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    hk = k.shape[1]
    if hk == 0 or hq == 0 or hq % hk:
        raise ValueError(f"packed_attention: {hq} query heads are not a multiple of {hk} key/value heads")
    if not packed_attention_supported(q):
        raise _lib.NF4Unsupported(_lib.NF4B_ERR_UNSUPPORTED,
                                  f"packed_attention: {q.dtype} head_dim {d} on {q.device} (fp16 or bf16 CUDA "
                                  "tensors, head_dim a multiple of 8 up to 128)")
    if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 1 or cu.device != q.device or not cu.is_contiguous():
        raise ValueError("packed_attention: cu must be a contiguous int32 vector of B + 1 row starts on q's device")
    left, right = (int(x) for x in window)
    if left < -1 or right < -1:
        raise ValueError(f"packed_attention: window {tuple(window)}: bounds are >= 0, or -1 for none")
    left, right = min(left, n), min(right, n)  # further than the longest sequence: no bound
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 2.0 ** -149 <= scale < 2.0 ** 127:  # (fp32, and so is scale log2(e))
        raise ValueError(f"packed_attention: scale must be positive and below 2^127, got {scale}")
    # (a forward-mode tangent goes there too, to be refused: the kernels on their own would drop it)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
            or _dual_level() and any(forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v))):
        return _PackedAttention.apply(q, k, v, cu, left, right, scale)
    return _attn_forward(q, k, v, cu, left, right, scale)[0]


# The backward's softmax - onehot is written as fp16 times this power of two (exact to divide
# out): a 151,936-entry row's probabilities are ~1e-5 and would otherwise sit in fp16's
# subnormal range.
CE_GRAD_SCALE = 1024.0


class _HeadCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, embed, labels):
        h2 = _c(h)
        logits = h2 @ embed.t()  # [rows, vocab] fp16 (cuBLAS)
        rows, vocab = logits.shape
        lab = _c(labels.to(torch.int64))
        loss = torch.empty(rows, dtype=torch.float32, device=h.device)
        lse = torch.empty(rows, dtype=torch.float32, device=h.device)
        _lib.check(_lib.lib().nf4b_ce_fwd(logits.data_ptr(), lab.data_ptr(), loss.data_ptr(), lse.data_ptr(),
                                          rows, vocab, _stream(h.device)), "nf4b_ce_fwd")
        ctx.save_for_backward(logits, lab, lse, embed)
        return loss.sum()

    @staticmethod
    def backward(ctx, g):
        logits, lab, lse, embed = ctx.saved_tensors
        rows, vocab = logits.shape
        gs = (g.float() * CE_GRAD_SCALE).reshape(1).contiguous()
        # softmax - onehot over the logits' own storage (they are not needed afterwards)
        _lib.check(_lib.lib().nf4b_ce_bwd(logits.data_ptr(), lab.data_ptr(), lse.data_ptr(), gs.data_ptr(),
                                          rows, vocab, _stream(logits.device)), "nf4b_ce_bwd")
        dh = logits @ embed
        dh.mul_(1.0 / CE_GRAD_SCALE)
        return dh, None, None


def head_cross_entropy(h: torch.Tensor, embed: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Sum over rows of CE(h @ embed^T, labels): fp16 logits from one GEMM, then the fused
    loss kernel; the gradient of h only (the embedding is frozen).  Labels outside
    [0, vocab) are ignored."""
    return _HeadCrossEntropy.apply(h, embed, labels)
