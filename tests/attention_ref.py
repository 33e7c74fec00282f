"""Packed-row attention and its gradients in 64 bits from the definition, with elementwise error
bounds for a kernel that rounds as attention.cu does."""
import torch


def row_mask(ln, left, right, device):
    i = torch.arange(ln, device=device)
    gap = i[None, :] - i[:, None]
    see = torch.ones(ln, ln, dtype=torch.bool, device=device)
    if left >= 0:
        see &= gap >= -left
    if right >= 0:
        see &= gap <= right
    return see


def reference(q, k, v, edges, left, right, scale, dout=None):
    """{name: (value, bound)} in float64 for out, and dq, dk, dv when dout is given.

    With h = eps / 2 of the type (half a step relative to a value) and t = 2e-5 for the 32-bit sums
    and exponentials (128-term dot products, |s| below ~100: |s| 2^-24 in the exponent, a few
    steps each), elementwise:
      out : p is rounded once before its product with v, out once:  h (|o| + P|V|) + t P|V|
      dv  : the same with P^T and |dO|
      ds  : its own rounding h |ds|, and do.o taken from the rounded o: h p (|dO|.|O|); 32 bits:
            t p (|dO|.|V| + |dO|.|O|)
      dq, dk : scale (that) |K|, |Q|, and the output's rounding h |dq|
    fp16 adds its smallest steps: 2^-25 for an output below its normal range, and 2^-25 of the row's
    largest probability for each p (P holds exp(s - max) with the maximum taken as 1)."""
    dt = q.dtype
    h = torch.finfo(dt).eps / 2
    t = 2e-5
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    q, k, v = q.double(), k.double(), v.double()
    n, hq, d = q.shape
    grp = hq // k.shape[1]
    z = torch.zeros_like
    res = {"out": (z(q), z(q))}
    if dout is not None:
        do_all = dout.double()
        res.update(dq=(z(q), z(q)), dk=(z(k), z(k)), dv=(z(k), z(k)))
    for a, b in zip(edges[:-1], edges[1:]):
        if a == b:
            continue
        see = row_mask(b - a, left, right, q.device)
        for hh in range(hq):
            g = hh // grp
            Q, K, V = q[a:b, hh], k[a:b, g], v[a:b, g]
            s = (Q @ K.T * scale).masked_fill(~see, float("-inf"))
            p = torch.softmax(s, -1)
            o = p @ V
            pv = p @ V.abs()
            res["out"][0][a:b, hh] = o
            res["out"][1][a:b, hh] = h * (o.abs() + pv) + t * pv + tiny * (1 + see.double() @ V.abs())
            if dout is None:
                continue
            dO = do_all[a:b, hh]
            dp = dO @ V.T
            delta = (dO * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            adelta = (dO.abs() * o.abs()).sum(-1, keepdim=True)
            eds = h * ds.abs() + p * h * adelta + t * p * (dO.abs() @ V.abs().T + adelta) + tiny * p * dO.abs().sum(-1, keepdim=True)
            res["dv"][0][a:b, g] += p.T @ dO
            res["dv"][1][a:b, g] += (h + t) * (p.T @ dO.abs()) + tiny * (see.double().T @ dO.abs())
            res["dq"][0][a:b, hh] = scale * ds @ K
            res["dq"][1][a:b, hh] = scale * eds @ K.abs()
            res["dk"][0][a:b, g] += scale * ds.T @ Q
            res["dk"][1][a:b, g] += scale * eds.T @ Q.abs()
    for name in ("dq", "dk", "dv"):
        if name in res:
            ref, bound = res[name]
            res[name] = (ref, bound + h * ref.abs() + tiny)
    return res


def assert_within(got, ref, bound, what):
    """Every element within its bound (x1.05 for the 64-bit bound's own first-order terms)."""
    err = (got.double() - ref).abs()
    bad = ~(err <= 1.05 * bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst error "
                                 f"{float(err[bad].max()) if bool(bad.any()) else 0:.3e} at "
                                 f"{bad.nonzero()[0].tolist()} (bound {float(bound[bad].max()):.3e})")
