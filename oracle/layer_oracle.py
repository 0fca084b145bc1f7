"""CPU restatement, in 64 bits and token by token, of the operators of a selective state space layer: the scan with a decay per
channel and state, the convolution that carries its history, the projection with its epilogue.  Test infrastructure only.

With `magnitude=True` the functions return, for every output, the sum of the magnitudes of the terms that it is made of: what a
rounding error of the summation is relative to."""
from __future__ import annotations

import torch

F = torch.nn.functional


def softplus(v):
    return F.softplus(v, threshold=200.0)


def selective_scan_ref(x, dt, A, B, C, D=None, z=None, init=None, *, dt_bias=None, dt_softplus=False, lengths=None, dy=None, dfinal=None,
                       magnitude=False):
    """dict of y, final_state and, with `dy`, the gradients by the reverse recurrence (no autograd)."""
    f = torch.float64
    mag = (lambda t: t.abs()) if magnitude else (lambda t: t)
    x, dt, A, B, C = (t.detach().to(f).cpu() for t in (x, dt, A, B, C))
    Bn, L, Dn = x.shape
    N = A.shape[1]
    B, C = (t.reshape(Bn, L, -1, N) for t in (B, C))
    G = B.shape[2]
    opt = lambda t: None if t is None else t.detach().to(f).cpu()
    D, z, init, dt_bias, dy, dfinal = (opt(t) for t in (D, z, init, dt_bias, dy, dfinal))
    live = torch.ones(Bn, L, 1, dtype=torch.bool) if lengths is None else \
        (torch.arange(L)[None, :] < lengths.cpu().clamp(0, L)[:, None])[..., None]
    zero = torch.zeros((), dtype=f)
    x, dt, z = (None if t is None else torch.where(live, t, zero) for t in (x, dt, z))
    Bh, Ch = (torch.where(live[..., None], mag(t.repeat_interleave(Dn // G, 2)), zero) for t in (B, C))
    x = mag(x)
    pre = dt if dt_bias is None else dt + dt_bias
    s = torch.where(live, softplus(pre) if dt_softplus else pre, zero)
    dsd = torch.sigmoid(pre) if dt_softplus else torch.ones_like(pre)
    Dv = torch.zeros(Dn, dtype=f) if D is None else mag(D)
    a = torch.exp(s[..., None] * A)
    h = torch.zeros(Bn, Dn, N, dtype=f) if init is None else mag(init)
    hs, y0 = [h], torch.empty_like(x)
    for t in range(L):
        h = a[:, t] * h + (s[:, t] * x[:, t])[..., None] * Bh[:, t]
        hs.append(h)
        y0[:, t] = (h * Ch[:, t]).sum(-1) + Dv * x[:, t]
    gate = torch.ones_like(x) if z is None else mag(F.silu(z))
    out = dict(y=torch.where(live, y0 * gate, zero), final_state=h)
    if dy is None:
        return out
    dy = mag(torch.where(live, dy, zero))
    sg = None if z is None else torch.sigmoid(z)
    if z is not None:
        out["dz"] = dy * y0 * mag(sg * (1 + z * (1 - sg)))
    dy0 = dy * gate
    Aw = mag(A)
    g = torch.zeros(Bn, Dn, N, dtype=f) if dfinal is None else mag(dfinal).clone()
    dx, ds = torch.empty_like(x), torch.empty_like(x)
    dB, dC, dA = torch.empty_like(Bh), torch.empty_like(Ch), torch.zeros_like(A)
    for t in range(L - 1, -1, -1):
        dC[:, t] = dy0[:, t][..., None] * hs[t + 1]
        g = g + dy0[:, t][..., None] * Ch[:, t]
        gB = (g * Bh[:, t]).sum(-1)
        dx[:, t] = s[:, t] * gB + Dv * dy0[:, t]
        dB[:, t] = g * (s[:, t] * x[:, t])[..., None]
        q = g * a[:, t] * hs[t]
        ds[:, t] = x[:, t] * gB + (q * Aw).sum(-1)
        dA += (q * s[:, t][..., None]).sum(0)
        g = g * a[:, t]
    ddt = torch.where(live, ds * dsd, zero)
    grp = lambda t: t.view(Bn, L, G, Dn // G, N).sum(3)
    out.update(dx=dx, ddt=ddt, dA=dA, dB=grp(torch.where(live[..., None], dB, zero)), dC=grp(torch.where(live[..., None], dC, zero)),
               dD=(dy0 * x).sum((0, 1)), ddt_bias=ddt.sum((0, 1)), dinit=g)
    return out


def conv_carry_ref(x, w, b=None, history=None, *, lengths=None, activation=True, dout=None, dnew=None, magnitude=False):
    """dict of out, history (the new one) and, with `dout`, din, dhistory, dweight, dbias."""
    f = torch.float64
    mag = (lambda t: t.abs()) if magnitude else (lambda t: t)
    x, w = (t.detach().to(f).cpu() for t in (x, w))
    Bn, L, Cn = x.shape
    K = w.shape[1]
    hist = torch.zeros(Bn, K - 1, Cn, dtype=f) if history is None else history.detach().to(f).cpu()
    n = torch.full((Bn,), L) if lengths is None else lengths.cpu().clamp(0, L)
    live = (torch.arange(L)[None, :] < n[:, None])[..., None]
    zero = torch.zeros((), dtype=f)
    ext = torch.cat([hist, torch.where(live, x, zero)], 1)
    bv = torch.zeros(Cn, dtype=f) if b is None else b.detach().to(f).cpu()
    pre = bv + sum(w[:, k] * ext[:, k:k + L] for k in range(K))
    premag = bv.abs() + sum(w[:, k].abs() * ext[:, k:k + L].abs() for k in range(K))
    sg = torch.sigmoid(pre)
    out = dict(out=torch.where(live, (pre * sg if activation else pre) if not magnitude else premag, zero),
               history=mag(torch.stack([ext[i, int(m):int(m) + K - 1] for i, m in enumerate(n)])))
    if dout is None:
        return out
    dact = sg * (1 + pre * (1 - sg)) if activation else torch.ones_like(pre)
    dpre = mag(torch.where(live, dout.detach().to(f).cpu(), zero)) * (dact if not magnitude else 1.0 + premag)   # |act''| <= 1
    e = mag(ext)
    dext = torch.zeros_like(ext)
    for k in range(K):
        dext[:, k:k + L] += mag(w[:, k]) * dpre
    if dnew is not None:
        for i, m in enumerate(n):
            dext[i, int(m):int(m) + K - 1] += mag(dnew[i].detach().to(f).cpu())
    out.update(din=dext[:, K - 1:], dhistory=dext[:, :K - 1], dbias=dpre.sum((0, 1)),
               dweight=torch.stack([(dpre * e[:, k:k + L]).sum((0, 1)) for k in range(K)], 1))
    return out


def act_ref(v, act):
    return {"none": v, "silu": F.silu(v), "softplus": softplus(v), "relu2": F.relu(v) ** 2}[act]


def dact_ref(v, act):
    s = torch.sigmoid(v)
    return {"none": torch.ones_like(v), "silu": s * (1 + v * (1 - s)), "softplus": s, "relu2": 2 * F.relu(v)}[act]


def linear_ref(x, w, b=None, r=None, *, act="none", dout=None):
    """dict of out, pre and, with `dout`, dx, dweight, dbias; plus the magnitudes that their sums are made of under *_mag."""
    f = torch.float64
    x, w = (t.detach().to(f).cpu() for t in (x, w))
    x = x.reshape(-1, x.shape[-1])
    N = w.shape[0]
    bv = torch.zeros(N, dtype=f) if b is None else b.detach().to(f).cpu()
    pre, pmag = x @ w.t() + bv, x.abs() @ w.abs().t() + bv.abs()
    rv = torch.zeros_like(pre) if r is None else r.detach().to(f).cpu().reshape(-1, N)
    o = dict(pre=pre, pre_mag=pmag, out=act_ref(pre, act) + rv, out_mag=rv.abs())
    if dout is None:
        return o
    g = dout.detach().to(f).cpu().reshape(-1, N)
    dpre = g * dact_ref(pre, act)
    o.update(dpre=dpre, g=g, dx=dpre @ w, dweight=dpre.t() @ x, dbias=dpre.sum(0))
    return o
