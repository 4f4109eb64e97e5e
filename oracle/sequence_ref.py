"""Plain float64 forms of the sequence operators (torch, any device): layer norm, linear attention with a decay per head,
attention with a sliding window and sinks, each with the magnitudes that its rounding errors are measured against.

``mag`` values are the same sums over absolute values: an error of relative size e in every factor or partial sum moves
the result by at most e times a small count times ``mag``."""
import math

import torch


def layer_norm(x, w, b, eps, dy=None):
    """y, and with dy also (dx, dw, db), in float64."""
    x = x.double()
    c = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    xh = c * r
    w = torch.ones(x.size(-1), dtype=torch.float64, device=x.device) if w is None else w.double()
    y = xh * w + (0.0 if b is None else b.double())
    if dy is None:
        return y
    dy = dy.double()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return y, dx, (dy * xh).flatten(0, -2).sum(0), dy.flatten(0, -2).sum(0)


def sequences(t, starts):
    """The (length, heads, dim) pieces of a dense or packed tensor."""
    if starts is None:
        return list(t)
    s = starts.tolist()
    return [t[a:b] for a, b in zip(s[:-1], s[1:])]


def _weights(n, a, device):
    t = torch.arange(n, dtype=torch.float64, device=device)
    gap = t[:, None] - t
    return torch.where(gap >= 0, torch.exp(a * gap.clamp(min=0)), 0.0), t


def decay_sequence(q, k, v, a, scale, state=None, do=None, dstate=None):
    """One sequence and head in float64.  Returns a dict: o, state, and with do: dq, dk, dv, dstate; mag_* beside each."""
    out = {}
    for pre in ('', 'mag_'):
        if pre:
            q, k, v = q.abs(), k.abs(), v.abs()
            scale, state = abs(scale), None if state is None else state.abs()
            do, dstate = None if do is None else do.abs(), None if dstate is None else dstate.abs()
        n, d = q.shape
        w, t = _weights(n, a, q.device)
        s0 = torch.zeros(d, d, dtype=torch.float64, device=q.device) if state is None else state
        before, after = torch.exp(a * (t + 1))[:, None], torch.exp(a * (n - 1 - t))[:, None]
        p = (q @ k.mT) * w * scale
        out[pre + 'o'] = p @ v + scale * before * (q @ s0)
        out[pre + 'state'] = math.exp(a * n) * s0 + (k * after).mT @ v
        if do is None:
            continue
        ds = torch.zeros_like(s0) if dstate is None else dstate
        g = (do @ v.mT) * w * scale
        out[pre + 'dq'] = g @ k + scale * before * (do @ s0.mT)
        out[pre + 'dk'] = g.mT @ q + after * (v @ ds.mT)
        out[pre + 'dv'] = p.mT @ do + after * (k @ ds)
        out[pre + 'dstate'] = math.exp(a * n) * ds + scale * (q * before).mT @ do
    return out


def visible(n, window, sinks, device):
    i = torch.arange(n, device=device)
    gap = i[:, None] - i
    return (gap >= 0) & ((gap < window) | (i < sinks))


def window_sequence(q, k, v, window, sinks, scale, do=None):
    """One sequence and query head in float64.  Returns a dict: o, and with do: dq, dk, dv; mag_* beside each, and `size`, the
    largest sum of absolute products behind a visible score."""
    n = q.size(0)
    see = visible(n, window, sinks, q.device)
    s = torch.where(see, scale * (q @ k.mT), -math.inf)
    p = torch.softmax(s, 1) if n else s
    out = {'o': p @ v, 'mag_o': p @ v.abs(), 'size': float((scale * (q.abs() @ k.abs().mT) * see).detach().max()) if n else 0.0}
    if do is not None:
        delta = (do * out['o']).sum(1, keepdim=True)
        ds = scale * p * (do @ v.mT - delta)
        mag = scale * p * (do.abs() @ v.abs().mT + (do.abs() * out['mag_o']).sum(1, keepdim=True))
        out.update(dq=ds @ k, dk=ds.mT @ q, dv=p.mT @ do, mag_dq=mag @ k.abs(), mag_dk=mag.mT @ q.abs(), mag_dv=p.mT @ do.abs())
    return out


def window_slot(pos, window, sinks):
    return pos if pos < sinks else sinks + (pos - sinks) % window
