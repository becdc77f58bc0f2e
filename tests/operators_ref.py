"""The device operators restated in 64 bits, one row after the other, with their gradients as formulas.

With `absolute` a sum of products is evaluated on the absolute values of its terms.  A computed sum whose terms went through
at most c roundings each is off by at most c * 2^-24 (to first order) times that - the bounds of the GPU tests."""
import torch


def sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _line(x, w, off, initial, s):
    """A history behind its window."""
    W = w.shape[1]
    head = initial[s] if initial is not None else torch.zeros(W - 1, x.shape[1], dtype=x.dtype, device=x.device)
    return torch.cat([head, x[off[s]:off[s + 1]]])


def conv(x, w, b, off, initial, silu, absolute=False):
    W, S = w.shape[1], len(off) - 1
    if absolute:
        x, w, b, initial = x.abs(), w.abs(), None if b is None else b.abs(), None if initial is None else initial.abs()
    y, fin = torch.zeros_like(x), torch.zeros(S, W - 1, x.shape[1], dtype=x.dtype, device=x.device)
    for s in range(S):
        line = _line(x, w, off, initial, s)
        for t in range(off[s], off[s + 1]):
            k = t - off[s]
            v = (line[k:k + W] * w.t()).sum(0) + (b if b is not None else 0)
            y[t] = v if absolute or not silu else v * sigmoid(v)
        fin[s] = line[len(line) - (W - 1):]
    return y, fin


def conv_gradient(dy, x, w, b, off, initial, silu, dfinal=None, absolute=False):
    """(dx, dw, db, dinitial); absolute: what the terms' absolute values add up to (with |d silu| <= 1.1)."""
    W, S = w.shape[1], len(off) - 1
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w[:, 0])
    di = torch.zeros(S, W - 1, x.shape[1], dtype=x.dtype, device=x.device)
    for s in range(S):
        line = _line(x, w, off, initial, s)
        dline = torch.zeros_like(line)
        for t in range(off[s], off[s + 1]):
            k = t - off[s]
            win = line[k:k + W]
            v = (win * w.t()).sum(0) + (b if b is not None else 0)
            g = sigmoid(v)
            d = dy[t] * (g * (1 + v * (1 - g)) if silu else 1)
            if absolute:
                # rounding of v enters d through |d2 silu| <= 0.5
                m = (win.abs() * w.t().abs()).sum(0) + (b.abs() if b is not None else 0)
                d = dy[t].abs() * (1.1 + 0.5 * m if silu else 1)
                win = win.abs()
            dline[k:k + W] += d * (w.t().abs() if absolute else w.t())
            dw += (d * win).t()
            db += d
        if dfinal is not None:
            dline[len(line) - (W - 1):] += dfinal[s].abs() if absolute else dfinal[s]
        di[s], dx[off[s]:off[s + 1]] = dline[:W - 1], dline[W - 1:]
    return dx, dw, db, di


def _terms(u, delta, A, B, C, D, z, bias, use_softplus):
    raw = delta + (bias if bias is not None else 0)
    dt = softplus(raw) if use_softplus else raw
    per = u.shape[1] // B.shape[1]
    return raw, dt, B.repeat_interleave(per, 1), C.repeat_interleave(per, 1)


def scan(u, delta, A, B, C, D, z, bias, initial, off, use_softplus=True, absolute=False):
    raw, dt, Be, Ce = _terms(u, delta, A, B, C, D, z, bias, use_softplus)
    ab = torch.abs if absolute else (lambda v: v)
    S, (ch, N) = len(off) - 1, A.shape
    y, fin = torch.zeros_like(u), torch.zeros(S, ch, N, dtype=u.dtype, device=u.device)
    for s in range(S):
        h = ab(initial[s]) if initial is not None else torch.zeros(ch, N, dtype=u.dtype, device=u.device)
        for t in range(off[s], off[s + 1]):
            h = torch.exp(dt[t][:, None] * A) * h + ab((dt[t] * u[t])[:, None] * Be[t])
            v = (h * ab(Ce[t])).sum(1) + (ab(D * u[t]) if D is not None else 0)
            y[t] = v * ab(z[t] * sigmoid(z[t])) if z is not None else v
        fin[s] = h
    return y, fin


def scan_gradient(dy, u, delta, A, B, C, D, z, bias, initial, off, dfinal=None, use_softplus=True, absolute=False):
    """A dict with an entry for every input; absolute: the terms' absolute values."""
    raw, dt, Be, Ce = _terms(u, delta, A, B, C, D, z, bias, use_softplus)
    ab = torch.abs if absolute else (lambda v: v)
    S, (ch, N), G = len(off) - 1, A.shape, B.shape[1]
    f = torch.zeros_like
    out = dict(u=f(u), delta=f(u), A=f(A), B=f(B), C=f(C), D=torch.zeros(ch, dtype=u.dtype, device=u.device), z=f(u), bias=torch.zeros(ch, dtype=u.dtype, device=u.device),
               initial=torch.zeros(S, ch, N, dtype=u.dtype, device=u.device))
    for s in range(S):
        h = ab(initial[s]) if initial is not None else torch.zeros(ch, N, dtype=u.dtype, device=u.device)
        hs = [h]
        for t in range(off[s], off[s + 1]):
            h = torch.exp(dt[t][:, None] * A) * h + ab((dt[t] * u[t])[:, None] * Be[t])
            hs.append(h)
        g = ab(dfinal[s]) if dfinal is not None else torch.zeros(ch, N, dtype=u.dtype, device=u.device)
        for t in range(off[s + 1] - 1, off[s] - 1, -1):
            k = t - off[s]
            inner = (hs[k + 1] * ab(Ce[t])).sum(1) + (ab(D * u[t]) if D is not None else 0)
            dys = dy[t]
            if z is not None:
                sg = sigmoid(z[t])
                dz = sg * (1 + z[t] * (1 - sg))
                out["z"][t] = ab(dy[t]) * inner * (dz.abs() + 0.5 if absolute else dz)   # (+ 0.5: d silu is itself a sum)
                dys = dy[t] * z[t] * sg
            dys = ab(dys)
            g = g + ab(Ce[t]) * dys[:, None]
            a = torch.exp(dt[t][:, None] * A)
            out["C"][t] = (hs[k + 1] * dys[:, None]).view(G, -1, N).sum(1)
            out["B"][t] = (g * ab(dt[t] * u[t])[:, None]).view(G, -1, N).sum(1)
            gB = (g * ab(Be[t])).sum(1)
            q = g * a * hs[k]
            d = ab(u[t]) * gB + (q * ab(A)).sum(1)
            if use_softplus:
                d = d * sigmoid(raw[t])
            out["delta"][t] = d
            out["u"][t] = ab(dt[t]) * gB + (ab(D) * dys if D is not None else 0)
            out["A"] += q * ab(dt[t])[:, None]
            out["D"] += dys * ab(u[t])
            out["bias"] += d
            g = a * g
        out["initial"][s] = g
    return out


def log_probabilities(s, items, scale):
    """(log p of the items, p, which rows take part)"""
    on = (items >= 0) & (items < s.shape[1]) & ~torch.isneginf(s).all(1)
    lp = torch.log_softmax(scale * torch.where(on[:, None], s, torch.zeros_like(s)), 1)
    at = torch.where(on, items, 0).long()
    return torch.where(on, lp.gather(1, at[:, None])[:, 0], torch.zeros_like(lp[:, 0])), lp.exp(), on, at


def _dscores(p, at, on, coef, scale):
    d = -coef[:, None] * p
    d[torch.arange(len(at)), at] += coef
    return torch.where((on & (coef != 0))[:, None], scale * d, torch.zeros_like(d))


def preference(s, items, off, refs, beta, smoothing, scale, w):
    lp, p, on, at = log_probabilities(s, items, scale)
    gain = torch.where(on, lp - (refs if refs is not None else 0), torch.zeros_like(lp))
    sums = torch.stack([gain[a:b].sum() for a, b in zip(off, off[1:])]) if len(off) > 1 else torch.zeros(0, dtype=s.dtype)
    m = beta * (sums[0::2] - sums[1::2])
    loss = torch.zeros_like(m)
    if smoothing < 1:
        loss = loss + (1 - smoothing) * softplus(-m)
    if smoothing > 0:
        loss = loss + smoothing * softplus(m)
    dm = beta * (smoothing - 1 / (1 + torch.exp(m)))
    coef = torch.zeros_like(lp)
    for k in range(len(off) - 1):
        coef[off[k]:off[k + 1]] = dm[k // 2] * (w[k // 2] if w is not None else 0) * (1 if k % 2 == 0 else -1)
    return dict(loss=loss, margin=m, logp=lp, coef=coef, p=p, dscores=_dscores(p, at, on, coef, scale))


def policy(s, items, old, adv, refs, lo, hi, kl_coef, scale, w):
    lp, p, on, at = log_probabilities(s, items, scale)
    r = torch.exp(lp - old)
    free, held = r * adv, r.clamp(1 - lo, 1 + hi) * adv
    loss, c = -torch.minimum(free, held), torch.where(free <= held, -free, torch.zeros_like(free))
    kl = torch.zeros_like(lp)
    if refs is not None:
        x = refs - lp
        kl = torch.expm1(x) - x
        loss, c = loss + kl_coef * kl, c - kl_coef * torch.expm1(x)
    z = torch.zeros_like(lp)
    coef = torch.where(on, c * (w if w is not None else 0), z)
    return dict(loss=torch.where(on, loss, z), kl=torch.where(on, kl, z), logp=lp, coef=coef, p=p, dscores=_dscores(p, at, on, coef, scale))
