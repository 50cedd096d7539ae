"""The state-space scan and the short causal filter in 64 bits, walked as they are defined.

Values and gradients are written as sums of products, so the same walk on absolute values gives the
magnitude that the roundings of a 32-bit evaluation are relative to (``magnitude=True``).
"""
import torch

F64 = torch.float64
U = 2.0 ** -24  # half a step of fp32


def sig(v):
    return 1 / (1 + torch.exp(-v))


def softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def live_mask(lengths, Bn, T):
    at = torch.arange(T)
    if lengths is None:
        return torch.ones(Bn, T, dtype=torch.bool)
    return at[None] < lengths[:, None]


def ssm(i, softplus_on, grads=None, magnitude=False):
    """i: dict of CPU tensors (x, delta, A, B, C and optionally D, z, delta_bias, h0, lengths; B, C are
    (B, G, N, T)).  grads: (dy, dlast or None).  Returns a dict of float64 tensors."""
    g = {k: v.to(F64) if v is not None and v.is_floating_point() else v for k, v in i.items()}
    x, A = g["x"], g["A"]
    Bn, D, T = x.shape
    G, N = g["B"].shape[1:3]
    live = live_mask(g.get("lengths"), Bn, T)
    m = live[:, None]
    zero = torch.zeros((), dtype=F64)
    raw = g["delta"] + (g["delta_bias"][:, None] if g.get("delta_bias") is not None else 0)
    raw = torch.where(m, raw, zero)
    dt = torch.where(m, softplus(raw) if softplus_on else raw, zero)
    x = torch.where(m, x, zero)
    Bt = torch.where(live[:, None, None], g["B"], zero).repeat_interleave(D // G, 1)   # (B, D, N, T)
    Ct = torch.where(live[:, None, None], g["C"], zero).repeat_interleave(D // G, 1)
    skip = g["D"] if g.get("D") is not None else torch.zeros(D, dtype=F64)
    z = torch.where(m, g["z"], zero) if g.get("z") is not None else None
    h0 = g["h0"] if g.get("h0") is not None else torch.zeros(Bn, D, N, dtype=F64)
    mag = (lambda t: t.abs()) if magnitude else (lambda t: t)
    x, Bt, Ct, skip, h0 = mag(x), mag(Bt), mag(Ct), mag(skip), mag(h0)
    dts = mag(dt)
    a = torch.exp(dt[:, :, None] * A[None, :, :, None])                                # (B, D, N, T)
    u = dts * x
    hs, h = [], h0
    for t in range(T):
        h = a[..., t] * h + u[:, :, t, None] * Bt[..., t]
        hs.append(h)
    H = torch.stack(hs, -1) if T else torch.zeros(Bn, D, N, 0, dtype=F64)
    y = (Ct * H).sum(2) + skip[:, None] * x
    gate = z * sig(z) if z is not None else torch.ones_like(y)
    gate = mag(gate)
    out = dict(y=torch.where(m, y * gate, zero), last=h)
    if grads is None:
        return out
    dy_out, dlast = grads[0].to(F64), grads[1]
    dy_out = mag(torch.where(m, dy_out, zero))
    dy = dy_out * gate
    if z is not None:
        s = sig(z)
        out["dz"] = dy_out * y * (s * (1 + z.abs()) if magnitude else s * (1 + z * (1 - s)))
    c = mag(dlast.to(F64)) if dlast is not None else torch.zeros_like(h0)
    Am = mag(A)
    dx, dd = torch.zeros_like(x), torch.zeros_like(x)
    dA = torch.zeros(D, N, dtype=F64)
    dB, dC = torch.zeros_like(g["B"]), torch.zeros_like(g["C"])
    per = D // G
    for t in range(T - 1, -1, -1):
        before = hs[t - 1] if t else h0
        gt = Ct[..., t] * dy[:, :, t, None] + c
        c = a[..., t] * gt
        q = c * before
        gB = (gt * Bt[..., t]).sum(-1)
        dx[..., t] = dts[..., t] * gB + skip * dy[..., t]
        dd[..., t] = (Am * q).sum(-1) + x[..., t] * gB
        dA += (dts[:, :, t, None] * q).sum(0)
        dB[..., t] = (gt * u[:, :, t, None]).view(Bn, G, per, N).sum(2)
        dC[..., t] = (hs[t] * dy[:, :, t, None]).view(Bn, G, per, N).sum(2)
    if softplus_on:
        dd = dd * sig(raw)
    dd, dx = torch.where(m, dd, zero), torch.where(m, dx, zero)
    dB, dC = (torch.where(live[:, None, None], v, zero) for v in (dB, dC))
    out.update(dx=dx, ddelta=dd, dA=dA, dB=dB, dC=dC, dD=(dy * x).sum((0, 2)), ddelta_bias=dd.sum((0, 2)), dh0=c)
    return out


def conv(i, silu_on, grads=None, magnitude=False):
    """i: dict of CPU tensors (x, w and optionally b, x0, lengths)."""
    g = {k: v.to(F64) if v is not None and v.is_floating_point() else v for k, v in i.items()}
    x, w = g["x"], g["w"]
    Bn, D, T = x.shape
    K = w.shape[1]
    live = live_mask(g.get("lengths"), Bn, T)
    m = live[:, None]
    zero = torch.zeros((), dtype=F64)
    mag = (lambda t: t.abs()) if magnitude else (lambda t: t)
    x0 = g["x0"] if g.get("x0") is not None else torch.zeros(Bn, D, K - 1, dtype=F64)
    b = g["b"] if g.get("b") is not None else torch.zeros(D, dtype=F64)
    true_ext = torch.cat([x0, torch.where(m, x, zero)], -1)
    ext = mag(true_ext)
    true_pre = b[:, None] + sum(w[:, k, None] * true_ext[..., k:k + T] for k in range(K)) + torch.zeros(Bn, D, T, dtype=F64)
    pre = mag(b)[:, None] + sum(mag(w)[:, k, None] * ext[..., k:k + T] for k in range(K)) + torch.zeros(Bn, D, T, dtype=F64)
    s = sig(true_pre)
    # |silu'| <= 1.1, so an error of the argument comes through with that factor at most
    y = (pre * (1.1 if magnitude else s)) if silu_on else pre
    ends = (g["lengths"] if g.get("lengths") is not None else torch.full((Bn,), T)).tolist()
    out = dict(y=torch.where(m, y, zero), last=torch.stack([ext[k, :, e:e + K - 1] for k, e in enumerate(ends)]) if Bn else ext[..., :K - 1])
    if grads is None:
        return out
    dy = mag(torch.where(m, grads[0].to(F64), zero))
    # |silu''| <= 1/2: the argument's error comes through with that factor
    dpre = dy * (1.1 + 0.5 * pre if magnitude else s * (1 + true_pre * (1 - s))) if silu_on else dy
    dext = torch.zeros(Bn, D, T + K - 1, dtype=F64)
    for k in range(K):
        dext[..., k:k + T] += mag(w)[:, k, None] * dpre
    if grads[1] is not None:
        for k, e in enumerate(ends):
            dext[k, :, e:e + K - 1] += mag(grads[1].to(F64))[k]
    out.update(dx=torch.where(m, dext[..., K - 1:], zero), dx0=dext[..., :K - 1],
               dw=torch.stack([(dpre * ext[..., k:k + T]).sum((0, 2)) for k in range(K)], 1), db=dpre.sum((0, 2)))
    return out
