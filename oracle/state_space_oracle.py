"""The state-space operators in 64 bits, token by token from their definitions, with their gradients: the oracle of
``tests/test_state_space.py`` and ``tests/test_gpu_state_space.py``.

A padded token is left out by keeping the tokens that are there (``present``), so that nothing it holds can reach a result.
``absolute=True`` evaluates every sum over the magnitudes of its terms, which is what a bound on rounding errors scales with."""
import torch


def present(mask, b, T):
    return [t for t in range(T) if mask is None or not bool(mask[b, t])]


def conv(x, weight, bias, state, mask, silu, g=None, g_state=None, absolute=False):
    """-> dict(y, state[, gx, gweight, gbias, gstate]); everything fp64.  state None: zeros."""
    T, B, D = x.shape
    W = weight.shape[1]
    state = torch.zeros(B, W - 1, D, dtype=x.dtype, device=x.device) if state is None else state
    bias = torch.zeros(D, dtype=x.dtype, device=x.device) if bias is None else bias
    mag = (lambda t: t.abs()) if absolute else (lambda t: t)
    out = dict(y=torch.zeros_like(x), state=torch.zeros_like(state), gx=torch.zeros_like(x), gweight=torch.zeros_like(weight),
               gbias=torch.zeros_like(bias), gstate=torch.zeros_like(state))
    for b in range(B):
        ts = present(mask, b, T)
        seq = torch.cat([state[b], x[ts, b]])                     # [W - 1 + n, D]
        n = len(ts)
        out["state"][b] = seq[n:n + W - 1]
        wins = torch.stack([seq[j:j + n] for j in range(W)], -1)  # [n, D, W]
        pre = (wins * weight).sum(-1) + bias
        sig = torch.sigmoid(pre)
        size = (mag(wins) * mag(weight)).sum(-1) + mag(bias)
        out["y"][ts, b] = size if absolute else (pre * sig if silu else pre)
        if g is None:
            continue
        slope = sig * (1 + pre * (1 - sig)) if silu else torch.ones_like(pre)
        gp = g[ts, b].abs() * (1 + size) if absolute else g[ts, b] * slope
        out["gweight"] += (gp.unsqueeze(-1) * mag(wins)).sum(0)
        out["gbias"] += gp.sum(0)
        gseq = torch.zeros_like(seq)
        for j in range(W):
            gseq[j:j + n] += gp * mag(weight[:, j])
        if g_state is not None:
            gseq[n:n + W - 1] += mag(g_state[b])
        out["gstate"][b] = gseq[:W - 1]
        out["gx"][ts, b] = gseq[W - 1:]
    return out


def scan(x, dt, a, b, c, d, dt_bias, s, mask, softplus, g=None, g_s=None, absolute=False):
    """-> dict(y, s[, gx, gdt, ga, gb, gc, gd, gbias, gs]); everything fp64."""
    T, B, D = x.shape
    G, N = b.shape[2:]
    mag = (lambda t: t.abs()) if absolute else (lambda t: t)
    zero = torch.zeros(D, dtype=x.dtype, device=x.device)
    d = zero if d is None else d
    raw = dt + (zero if dt_bias is None else dt_bias)
    delta_of = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    wide = lambda t: t.repeat_interleave(D // G, 0)               # [G, N] -> [D, N]
    out = dict(y=torch.zeros_like(x), s=torch.zeros(B, D, N, dtype=x.dtype, device=x.device))
    if g is not None:
        out.update(gx=torch.zeros_like(x), gdt=torch.zeros_like(x), ga=torch.zeros_like(a), gb=torch.zeros_like(b), gc=torch.zeros_like(c),
                   gd=torch.zeros_like(zero), gbias=torch.zeros_like(zero), gs=torch.zeros_like(out["s"]))
    for i in range(B):
        ts = present(mask, i, T)
        st = torch.zeros(D, N, dtype=x.dtype, device=x.device) if s is None else mag(s[i])
        states = [st]
        for t in ts:
            st = torch.exp(delta_of[t, i, :, None] * a) * st + mag(delta_of[t, i] * x[t, i])[:, None] * mag(wide(b[t, i]))
            states.append(st)
            out["y"][t, i] = (mag(wide(c[t, i])) * st).sum(-1) + mag(d * x[t, i])
        out["s"][i] = st
        if g is None:
            continue
        G_ = torch.zeros_like(st) if g_s is None else mag(g_s[i])
        for k in reversed(range(len(ts))):
            t = ts[k]
            delta, xt, gt, bt, ct = delta_of[t, i], mag(x[t, i]), mag(g[t, i]), mag(wide(b[t, i])), mag(wide(c[t, i]))
            G_ = G_ + ct * gt[:, None]
            decay = torch.exp(delta[:, None] * a)
            p = G_ * decay * states[k]
            over = (G_ * bt).sum(-1)
            out["gc"][t, i] = (states[k + 1] * gt[:, None]).unflatten(0, (G, -1)).sum(1)
            out["gb"][t, i] = (G_ * (mag(delta) * xt)[:, None]).unflatten(0, (G, -1)).sum(1)
            out["gx"][t, i] = mag(delta) * over + mag(d) * gt
            out["ga"] += mag(delta)[:, None] * p
            out["gd"] += xt * gt
            graw = ((p * mag(a)).sum(-1) + xt * over) * slope[t, i]
            out["gdt"][t, i] = graw
            out["gbias"] += graw
            G_ = G_ * decay
        out["gs"][i] = G_
    return out


def norm(x, groups, weight, bias, gate, silu, eps, g=None, absolute=False):
    """-> dict(y[, gx, gweight, gbias, ggate]); everything fp64.  With ``absolute``, magnitudes times the condition
    1 + max |x| / deviation of the group, from which the subtraction of the mean loses bits."""
    C = x.shape[-1]
    weight = torch.ones(C, dtype=x.dtype, device=x.device) if weight is None else weight
    bias = torch.zeros(C, dtype=x.dtype, device=x.device) if bias is None else bias
    rows = lambda t: t.reshape(-1, groups, C // groups)
    xg, w, bb = rows(x), weight.view(groups, -1), bias.view(groups, -1)
    mean = xg.mean(-1, keepdim=True)
    dev = ((xg - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xn = (xg - mean) / dev
    n = xn * w + bb
    by = n if gate is None else rows(gate)
    sig = torch.sigmoid(by) if silu else torch.ones_like(by)
    act = by * sig
    slope = sig * (1 + by * (1 - sig)) if silu else torch.ones_like(by)
    if absolute:
        cond = 1 + xg.abs().amax(-1, keepdim=True) / dev
        n, xn = (1 + xn.abs()) * w.abs() + bb.abs(), 1 + xn.abs()
        act, slope = act.abs() + by.abs(), torch.full_like(slope, 1.1)
        if gate is None:
            act = act + n
    out = dict(y=n * act if gate is not None else act)
    if g is not None:
        gr = rows(g).abs() if absolute else rows(g)
        gn = gr * (act if gate is not None else (slope * (1 + n) if absolute else slope))
        h = gn * (w.abs() if absolute else w)
        if absolute:
            gx = (h + h.mean(-1, keepdim=True) + xn * (h * xn).mean(-1, keepdim=True)) / dev * cond
            gw, out["ggate"] = (gn * xn * cond).sum(0), gr * n * slope * (1 + by.abs()) * cond
        else:
            gx = (h - h.mean(-1, keepdim=True) - xn * (h * xn).mean(-1, keepdim=True)) / dev
            gw, out["ggate"] = (gn * xn).sum(0), gr * n * slope
        out.update(gx=gx, gweight=gw.flatten(), gbias=(gn * cond if absolute else gn).sum(0).flatten())
    if absolute:
        out["y"] = out["y"] * cond
    return {k: v.reshape(x.shape) if k in ("y", "gx", "ggate") else v for k, v in out.items()}
