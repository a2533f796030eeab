"""Float64 statements (CPU torch) of the attention of any range and of the query and key preparation, with bounds on the
rounding errors that a kernel with 16-bit operands may make.

attention():  s = scale q k^T, capped by a tanh, minus slope x distance, softmax over the visible keys, times v; the gradients
by the chain rule.  `u` is half a step of the operands' type.  The bounds, per element, count

    out   the probabilities rounded once and the result once:       u (P |V|) + u |out|
    dv    the probabilities and the result:                         u (P^T |dO|) + u |dv|
    dq    dS rounded, delta from the rounded output, the result:    u scale (|dS| + P delta') |K| + u |dq|,
          delta' = rowsum |dO o out|;  dk alike
and 32-bit sums: a dot product over D values is off by D 2^-24 of its absolute sum at most, which moves a probability by that
much of itself (times the scale) and dS by that much of P (|dO| |V|^T + delta').

A capped score may be off by 2^-21 of the cap; with `strict` by 2^-20 of itself and no more, however far the cap is.  In fp16 small
probabilities and dS lose bits, by half a step of 2^-24 each; with `strict` that step counts from the largest dS of a query (for dq) or of a key (for
dk) at 2^10, P for dv from 1 at 2^14 and for the output from a row's largest at 2^7, and delta is off by what the probabilities' rounding does to the output and its own two roundings leave.
"""
import torch


def positions(Tq, Tk, lens, B):
    n = torch.full((B,), Tk) if lens is None else lens.long()
    return n.unsqueeze(-1) - Tq + torch.arange(Tq)


def visible(B, Tq, Tk, causal=True, window=None, docs=None, prefix=None, lens=None):
    """(B, Tq, Tk) bool, and the distances i - j."""
    i = positions(Tq, Tk, lens, B).unsqueeze(-1)
    j = torch.arange(Tk)
    d = i - j
    W = window if window is not None else 1 << 60
    ok = ((d >= 0) & (d < W)) if causal else (d.abs() < W)
    if prefix is not None:
        ok = ok | (j < prefix.view(-1, 1, 1))
    if docs is not None:
        dq = docs[:, Tk - Tq:]
        ok = ok & (dq.unsqueeze(-1) == docs.unsqueeze(1)) & (dq >= 0).unsqueeze(-1)
    if lens is not None:
        ok = ok & (j < lens.view(-1, 1, 1)) & (i >= 0)
    return ok, d


def attention(q, k, v, scale=None, causal=True, window=None, cap=None, slopes=None, docs=None, prefix=None, lens=None,
              dout=None, u=0.0, strict=False):
    """{"out": (value, bound)} and with dout also dq, dk, dv; all (B, H, T, D) float64."""
    B, Hq, Tq, D = q.shape
    Hk, Tk = k.shape[1:3]
    R = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double().repeat_interleave(R, 1), v.double().repeat_interleave(R, 1)
    ok, dist = visible(B, Tq, Tk, causal, window, docs, prefix, lens)
    ok = ok.unsqueeze(1)
    used = ok.any(-2)                                    # keys that nobody sees count as zeros, whatever they hold
    k, v = (torch.where(used.expand(B, Hq, Tk).unsqueeze(-1), x, 0.0) for x in (k, v))
    q = torch.where(ok.any(-1).expand(B, Hq, Tq).unsqueeze(-1), q, 0.0)
    raw = scale * (q @ k.transpose(-1, -2))
    th = torch.tanh(raw / cap) if cap else None
    s = cap * th if cap else raw
    tanh_err = 0.0 if not cap else 2.0 ** -20 * s.abs() if strict else 2.0 ** -21 * cap
    if slopes is not None:
        s = s - slopes.double().view(-1, 1, 1) * dist.abs().double().unsqueeze(1)
    s = torch.where(ok, s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.where(ok, torch.exp(s - torch.where(m.isinf(), 0.0, m)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = p @ v
    f = D * 2.0 ** -24
    # how far a probability may be off, relative: its score's absolute sum, the exponential's argument (2^-23 of it), both for
    # the score and for the row's log-sum-exp; and what the cap's tanh is off by
    amp = f * (abs(scale) if strict else scale) * (q.abs() @ k.abs().transpose(-1, -2)) + 2.0 ** -21 * torch.where(ok, s, 0.0).abs() + tanh_err
    if strict and cap:                                   # a capped score is off by the cap's range at most
        amp = amp.clamp_max(2.0 * cap)
    amp = torch.where(ok, amp, 0.0)
    amp = 1.05 * (amp + amp.amax(-1, keepdim=True)) + 2.0 ** -18
    half = u < 2.0 ** -9 and u > 0                       # fp16: probabilities below 2^-14 of the row's largest lose bits
    sub = 2.0 ** -24 if half else 0.0
    # a result below 2^-14 is rounded to a multiple of fp16's smallest step, 2^-24: off by half of it
    tiny = 2.0 ** -30 if u == 0 else 2.0 ** -25 if half else 0.0
    a = p @ v.abs()
    res = {"out": (out, u * (a + out.abs()) * 1.02 + (p * amp) @ v.abs() + sub * ok.double() @ v.abs() + tiny)}
    if strict and half:
        few = 2.0 ** -32 * p.amax(-1, keepdim=True) * ok.double()
        res["out"] = (out, u * (a + out.abs()) * 1.02 + (p * amp + few) @ v.abs() + tiny)
    if dout is None:
        return res
    g = torch.where(ok.any(-1).expand(B, Hq, Tq).unsqueeze(-1), dout.double(), 0.0)
    dp = g @ v.transpose(-1, -2)
    delta = (g * out).sum(-1, keepdim=True)
    tang = (1.0 - th * th) if cap else torch.ones((), dtype=torch.float64)
    ds = p * (dp - delta) * tang
    share = lambda x: x.reshape(B, Hk, R, *x.shape[2:]).sum(2)
    dq, dk, dv = scale * (ds @ k), scale * share(ds.transpose(-1, -2) @ q), share(p.transpose(-1, -2) @ g)
    d1 = (g.abs() * out.abs()).sum(-1, keepdim=True)
    pa = g.abs() @ v.abs().transpose(-1, -2)
    # an error of the score moves 1 - tanh^2 by at most twice it over the cap
    e = u * (1.02 * ds.abs() + p * (1.02 * d1)) + p * (f * (pa + d1) + (amp + (2 * amp / cap if cap else 0.0)) * (dp.abs() + d1)) \
        + u * sub * ok.double()
    if half:
        e = e + sub * ok.double()
    sc = abs(scale)
    res["dq"] = (dq, sc * (e @ k.abs()) + u * dq.abs() * 1.02 + tiny)
    res["dk"] = (dk, share(sc * (e.transpose(-1, -2) @ q.abs())) + u * dk.abs() * 1.02 + tiny)
    ep = p * (u * 1.02 + amp) + sub * ok.double()
    if strict:
        step = 2.0 ** -25 if half else 0.0
        d = ok.double()
        # delta is formed from the output, in which each probability was rounded: off by u sum_j p_j |dp_j|
        e0 = u * 1.02 * (ds.abs() + p * (p * dp.abs()).sum(-1, keepdim=True)) + p * (2 * u * u * d1 + step * g.abs().sum(-1, keepdim=True)
                                        + f * (pa + d1) + (amp + (2 * amp / cap if cap else 0.0)) * (dp.abs() + d1))
        at = lambda dim: step * 2.0 ** -10 * d * ds.abs().amax(dim, keepdim=True)
        res["dq"] = (dq, sc * ((e0 + at(-1)) @ k.abs()) + u * dq.abs() * 1.02 + tiny)
        # (heads that share a key share its power of two)
        top = share(ds.abs().amax(-2, keepdim=True)).repeat_interleave(R, 1) if R > 1 else ds.abs().amax(-2, keepdim=True)
        e1 = e0 + step * 2.0 ** -10 * d * top
        res["dk"] = (dk, share(sc * (e1.transpose(-1, -2) @ q.abs())) + u * dk.abs() * 1.02 + tiny)
        ep = p * (u * 1.02 + amp) + step * 2.0 ** -14 * d
    res["dv"] = (dv, share(ep.transpose(-1, -2) @ g.abs()) + u * dv.abs() * 1.02 + tiny)
    return res


def rope(x, w, freqs, pos, eps=1e-6, interleaved=False, dy=None):
    """Normed and rotated rows of x (B, H, T, D) at positions pos (B or 1, T); with dy also dx and dw."""
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    r = 2 * freqs.numel()
    ang = pos.double().unsqueeze(-1) * freqs.double()
    cos, sin = torch.cos(ang).unsqueeze(1), torch.sin(ang).unsqueeze(1)
    sl = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))

    def turn(y, sn):
        o = y.clone()
        a, b = y[..., sl[0]], y[..., sl[1]]
        o[..., sl[0]], o[..., sl[1]] = a * cos - b * sn, b * cos + a * sn
        return o

    rr = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * rr
    y = turn(n * w, sin)
    if dy is None:
        return y
    g = turn(dy.double(), -sin)
    h = g * w
    return y, rr * (h - n * (h * n).mean(-1, keepdim=True)), (g * n).sum((0, 1, 2)), (g * n).abs().sum((0, 1, 2))
