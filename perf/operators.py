"""Measured cases of the training step's attention over packed rows (forward, and forward with
backward) and of the gradient list's global norm and clipping.

Packed attention: q [N, Hq, D], k/v [N, Hk, D] hold B token sequences one after the other,
sequence b in rows [cu[b], cu[b+1]); inside a sequence token i sees the tokens j with
i - left <= j <= i + right (a negative bound is no bound; (-1, 0) is causal), query head h reads
key/value head h // (Hq / Hk):
    s_ij = scale q_i.k_j,  p_ij = exp(s_ij) / sum_j exp(s_ij),  o_i = sum_j p_ij v_j
    dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i.v_j - do_i.o_i),
    dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
(k/v gradients summed over the query heads that share them); rows behind cu[B] give zeros.

Clipping: g' = (g / divisor) min(1, max_norm / (norm + 1e-6)), norm the 2-norm of all g / divisor.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# (out, in) of one layer's projections q, k, v, o, gate, up, down
LAYER = ((1536, 1536), (256, 1536), (256, 1536), (1536, 1536), (8960, 1536), (8960, 1536), (1536, 8960))


def _attn(name, train, tokens, rows, **kw):
    c = {"name": name, "op": "attention", "train": train, "tokens": tokens, "rows": rows, "heads": 12, "kv_heads": 2,
         "head_dim": 128, "dtype": "fp16", "left": -1, "right": 0, "spread": 0.86, "pad": 0, "fused": False, "lens": 1}
    c.update(kw)
    return c


def _clip(name, kind, count, dtype, max_norm, divisor, lens=1):
    return {"name": name, "op": "clip", "kind": kind, "count": count, "dtype": dtype, "max_norm": max_norm,
            "divisor": divisor, "lens": lens}


def listed():
    return [
        # a handful of short rows (an evaluation batch's stragglers): launch latency is all there is
        _attn("fwd 63 tokens", False, 63, 3),
        # the QLoRA step: 4 rows of up to 512 with 1,170 real tokens, packed
        _attn("fwd step 1170", False, 1170, 4),
        # bidirectional encoder rows of odd lengths, one key/value head per query head, q/k/v as
        # slices of one projection output, a padded token buffer
        _attn("fwd bf16 d64 full 4099", False, 4099, 9, heads=16, kv_heads=16, head_dim=64, dtype="bf16", right=-1, pad=61,
              fused=True),
        # one long document: the largest forward
        _attn("fwd long 16384", False, 16384, 1, spread=0.0),
        _attn("train 63 tokens", True, 63, 3),
        # one layer's attention in the QLoRA step, forward and backward
        _attn("train step 1170", True, 1170, 4),
        # a larger batch with a sliding window, bf16
        _attn("train bf16 window 8192", True, 8192, 16, dtype="bf16", left=255, fused=True),
        # one long document, forward and backward
        _attn("train long 8192", True, 8192, 1, spread=0.0),
        # one layer's q and v adapters
        _clip("clip 1 layer", "adapter", 1, "fp32", 1.0, 1166.0),
        # the QLoRA step's 112 adapter gradients, divided by the labelled-token count on the way
        _clip("clip 28 layers", "adapter", 28, "fp32", 0.3, 1166.0),
        # tensors of odd sizes (biases, norms, adapters of other ranks), fp16, under the limit
        _clip("clip odd fp16", "odd", 61, "fp16", 1e6, 0.0),
        # full fine-tuning: the weight gradients of four layers' projections, bf16
        _clip("clip weights bf16", "weights", 4, "bf16", 1.0, 0.0),
    ]


def draw(rng):
    if rng.random() < 0.3:
        kind = rng.choice(["adapter", "odd", "weights"])
        count = {"adapter": rng.randint(1, 40), "odd": rng.randint(1, 200), "weights": rng.randint(1, 3)}[kind]
        c = _clip("", kind, count, rng.choice(["fp32", "fp16", "bf16"]), rng.choice([0.1, 1.0, 10.0, 1e6]),
                  rng.choice([0.0, float(rng.randint(1, 5000))]), rng.randint(0, 1 << 30))
        if kind == "weights" and c["dtype"] == "fp32":
            c["count"] = min(c["count"], 2)
    else:
        train = rng.random() < 0.6
        heads, kv = rng.choice([(12, 2), (12, 2), (16, 16), (8, 8), (16, 4), (6, 1), (14, 2)])
        tokens = int(math.exp(rng.uniform(math.log(16), math.log(8192 if heads <= 12 else 4096))))
        rows = min(tokens, int(math.exp(rng.uniform(0, math.log(24)))))
        window = rng.choice([(-1, 0), (-1, 0), (-1, -1), (rng.randint(0, 600), 0), (rng.randint(0, 300), rng.randint(0, 300))])
        if window == (-1, -1) and tokens > 4096:
            window = (-1, 0)
        c = _attn("", train, tokens, rows, heads=heads, kv_heads=kv, head_dim=rng.choice([128, 128, 64, 96, 80]),
                  dtype=rng.choice(["fp16", "bf16"]), left=window[0], right=window[1], spread=rng.choice([0.0, 0.86, 0.99]),
                  pad=rng.choice([0, 0, rng.randint(1, 130)]), fused=rng.random() < 0.4, lens=rng.randint(0, 1 << 30))
    del c["name"]
    return c


def lengths(case):
    """The rows' lengths: `tokens` shared out over `rows` rows, by weights in [1 - spread, 1]."""
    r = random.Random(case["lens"])
    n, b = case["tokens"], case["rows"]
    w = [1.0 - case["spread"] * r.random() for _ in range(b)]
    edge = [round((n - b) * sum(w[:i]) / sum(w)) + i for i in range(b + 1)]
    return [edge[i + 1] - edge[i] for i in range(b)]


def sizes(case):
    """The gradients' shapes."""
    if case["kind"] == "adapter":
        return [(16, 1536), (1536, 16), (16, 1536), (256, 16)] * case["count"]
    if case["kind"] == "weights":
        return list(LAYER) * case["count"]
    r = random.Random(case["lens"])
    return [(int(math.exp(r.uniform(0, math.log(60000)))),) for _ in range(case["count"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "clip":
        shapes = sizes(case)
        numel = [math.prod(s) for s in shapes]
        flat = torch.randn(sum(numel), device="cuda", generator=g, dtype=torch.float32)
        flat = flat.mul_(1e-2 if case["divisor"] == 0.0 else 1.0).to(dt)
        out = torch.empty_like(flat)
        return {"case": case, "grads": [v.view(s) for v, s in zip(flat.split(numel), shapes)], "out": out,
                "outs": [v.view(s) for v, s in zip(out.split(numel), shapes)],
                "divisor": None if case["divisor"] == 0.0 else torch.full((1,), case["divisor"], device="cuda")}
    lens = lengths(case)
    n, hq, hk, d = case["tokens"] + case["pad"], case["heads"], case["kv_heads"], case["head_dim"]
    x = torch.randn(n, hq + 2 * hk, d, device="cuda", generator=g).to(dt)
    q, k, v = x.split([hq, hk, hk], dim=1)
    if not case["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
    s = {"case": case, "q": q, "k": k, "v": v, "cu": cu, "longest": max(lens), "window": (case["left"], case["right"])}
    if case["train"]:
        s["dout"] = (torch.randn(n, hq, d, device="cuda", generator=g) * 0.02).to(dt)
    return s


def run(state):
    if state["case"]["op"] == "clip":
        return _run_clip(state)
    if own:
        from stew_b200.step_ops import packed_attention
        if not state["case"]["train"]:
            with torch.no_grad():
                return packed_attention(state["q"], state["k"], state["v"], state["cu"], window=state["window"])
        leaves = [state[t].detach().requires_grad_(True) for t in ("q", "k", "v")]
        o = packed_attention(*leaves, state["cu"], window=state["window"])
        return (o.detach(), *torch.autograd.grad(o, leaves, state["dout"]))
    return _plain_attention(state)


def _run_clip(s):
    case = s["case"]
    if own:
        from stew_b200.dp import clip_grads
        norm = clip_grads(s["grads"], case["max_norm"], divisor=s["divisor"], out=s["outs"])
        return norm, s["out"]
    x = torch.cat([t.reshape(-1) for t in s["grads"]]).float()
    if s["divisor"] is not None:
        x = x / s["divisor"]
    norm = x.double().square().sum().sqrt()
    c = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return norm.float(), (x * c).to(DTYPES[case["dtype"]])


def _plain_attention(s):
    """The sequences as a padded batch [B, L], 32-bit products and sums."""
    case, q, k, v, cu = s["case"], s["q"], s["k"], s["v"], s["cu"].long()
    dev, (n, hq, d), hk, big = q.device, q.shape, k.shape[1], s["longest"]
    grp, scale = hq // hk, 1.0 / math.sqrt(d)
    at = torch.arange(big, device=dev)
    real = at[None, :] < (cu[1:] - cu[:-1])[:, None]                       # [B, L]
    idx = (cu[:-1, None] + at[None, :]).clamp(max=n - 1)
    tok = torch.arange(n, device=dev)
    row = torch.searchsorted(cu[1:], tok, right=True).clamp(max=cu.numel() - 2)
    pos = (tok - cu[row]).clamp(max=big - 1)
    inside = (tok < cu[-1])[:, None, None]

    def padded(x, groups):  # [N, H, D] -> [B, Hk, groups, L, D], zeros behind each sequence's end
        y = torch.where(real[:, :, None, None], x[idx].float(), 0.0)
        return y.view(y.shape[0], big, hk, groups, d).permute(0, 2, 3, 1, 4)

    def packed(y, dt):      # [B, Hk, groups, L, D] -> [N, H, D]
        y = y.permute(0, 3, 1, 2, 4).reshape(y.shape[0], big, -1, d)
        return torch.where(inside, y[row, pos], 0.0).to(dt)

    see = real[:, None, :].expand(-1, big, -1)
    if s["window"][0] >= 0:
        see = see & (at[None, None, :] >= at[None, :, None] - s["window"][0])
    if s["window"][1] >= 0:
        see = see & (at[None, None, :] <= at[None, :, None] + s["window"][1])
    see = see[:, None, None]
    qp, kp, vp = padded(q, grp), padded(k, 1), padded(v, 1)
    p = (qp * scale) @ kp.transpose(-1, -2)
    p = p.masked_fill_(~see, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = p @ vp
    out = packed(o, q.dtype)
    if not case["train"]:
        return out
    dop = padded(s["dout"], grp)
    dv = (p.transpose(-1, -2) @ dop).sum(2, keepdim=True)
    ds = dop @ vp.transpose(-1, -2)
    ds = ds.sub_((dop * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ kp
    dk = (ds.transpose(-1, -2) @ qp).sum(2, keepdim=True)
    return out, packed(dq, q.dtype), packed(dk, q.dtype), packed(dv, q.dtype)


def _pairs(case):
    """Visible (query, key) pairs over all rows."""
    total = 0
    for ln in lengths(case):
        i = np.arange(ln, dtype=np.int64)
        lo = np.maximum(i - case["left"], 0) if case["left"] >= 0 else np.zeros_like(i)
        hi = np.minimum(i + case["right"], ln - 1) if case["right"] >= 0 else np.full_like(i, ln - 1)
        total += int((hi - lo + 1).sum())
    return total


def work(case):
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in sizes(case))
        return {"bytes": 2 * n * (4 if case["dtype"] == "fp32" else 2) + 4, "flops": 4 * n}
    n, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    q, kv, mac = n * hq * d * 2, n * hk * d * 2, 2 * _pairs(case) * hq * d
    if not case["train"]:
        return {"bytes": 2 * q + 2 * kv, "flops": 2 * mac}
    return {"bytes": 4 * q + 4 * kv, "flops": 7 * mac}


def exact(case, seed):
    """The definition in 64 bits, one sequence and one key/value head at a time."""
    s = prepare(case, seed)
    if case["op"] == "clip":
        g = [t.double() for t in s["grads"]]
        if case["divisor"] != 0.0:
            g = [t / case["divisor"] for t in g]
        norm = math.sqrt(sum(float(torch.linalg.vector_norm(t)) ** 2 for t in g))
        c = min(1.0, case["max_norm"] / (norm + 1e-6))
        return torch.tensor(norm, dtype=torch.float64), torch.cat([(t * c).reshape(-1) for t in g])
    q, k, v = (s[t].double() for t in ("q", "k", "v"))
    scale, grp = case["head_dim"] ** -0.5, case["heads"] // case["kv_heads"]
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a = 0
    for ln in lengths(case):
        b = a + ln
        i = torch.arange(ln, device=q.device)
        gap = i[None, :] - i[:, None]
        hide = torch.zeros(ln, ln, dtype=torch.bool, device=q.device)
        if case["left"] >= 0:
            hide |= gap < -case["left"]
        if case["right"] >= 0:
            hide |= gap > case["right"]
        for h in range(case["heads"]):
            kh, vh = k[a:b, h // grp], v[a:b, h // grp]
            p = torch.softmax((q[a:b, h] @ kh.T * scale).masked_fill(hide, -math.inf), -1)
            out[a:b, h] = p @ vh
            if case["train"]:
                do = s["dout"][a:b, h].double()
                dv[a:b, h // grp] += p.T @ do
                dp = do @ vh.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[a:b, h] = ds @ kh
                dk[a:b, h // grp] += ds.T @ q[a:b, h]
        a = b
    return (out, dq, dk, dv) if case["train"] else out
