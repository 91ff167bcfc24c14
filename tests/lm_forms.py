"""Plain statements in 64 bits of the masked attention and of the paged 8-bit cache, with what rounding may do to them.

masked() returns o, dq, dk, dv and, for each, the sum of the magnitudes of its terms: a result computed in float32 from inputs
of a type whose half step is u = finfo.eps / 2, and rounded once to that type, is off by at most

    u * |result| + u * terms + F * terms

The first part is the output's rounding.  The second is there for 16-bit inputs: a weight p (or the gradient of a score) that
goes through a matrix instruction is rounded to the type, relative error u a term; D = sum do*o in the backward is formed from
the rounded o, which moves each score gradient by at most p * u * sum |do*o| (in `terms` of dq and dk).  F = 2^-24 * (3 W + 64):
a distance is a sum of W terms (relative error W 2^-24 in any order), a logit of magnitude L <= 20 in these tests moves by
W 2^-24 L / W-th of that on average and exp turns it into a relative error of p; the sums over tokens add 2^-24 a partial sum."""
import math

import torch


def visible(T, S, B, causal, doc, prefix):
    i = torch.arange(S - T, S)
    s = torch.arange(S)
    see = torch.ones(B, T, S, dtype=torch.bool)
    if causal:
        see &= s[None] <= i[:, None]
        if prefix is not None:
            see |= s[None, None] < prefix[:, None, None].long()
    if doc is not None:
        see &= (doc[:, i][:, :, None] == doc[:, None, :]) & (doc[:, i][:, :, None] >= 0)
    return see


def masked(q, k, v, do=None, doc=None, prefix=None, causal=True, cap=0.0, slopes=None):
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    doc = None if doc is None else doc.cpu()
    prefix = None if prefix is None else prefix.cpu()
    B, T, H, W = q.shape
    S, Hk, Wv = k.shape[1], k.shape[2], v.shape[3]
    G = H // Hk
    see = visible(T, S, B, causal, doc, prefix)
    # what is hidden has no influence: rows that no one sees are taken as zero, whatever they hold
    seen = see.any(1)
    k = torch.where(seen[:, :, None, None], k, torch.zeros_like(k))
    v = torch.where(seen[:, :, None, None], v, torch.zeros_like(v))
    sees = see.any(2)
    q = torch.where(sees[:, :, None, None], q, torch.zeros_like(q))
    kk, vv = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    rw = 1 / math.sqrt(W)
    o = torch.zeros(B, T, H, Wv, dtype=torch.float64)
    to = torch.zeros_like(o)
    if do is not None:
        do = do.double().cpu()
        dq, tq = torch.zeros_like(q), torch.zeros_like(q)
        dkk, tkk = torch.zeros_like(kk), torch.zeros_like(kk)
        dvv, tvv = torch.zeros_like(vv), torch.zeros_like(vv)
    dist = (torch.arange(S - T, S)[:, None] - torch.arange(S)[None]).abs().double()
    for b in range(B):
        for h in range(H):
            d = q[b, :, None, h] - kk[b, None, :, h]
            a = -rw * d.abs().sum(-1)
            c = cap * torch.tanh(a / cap) if cap else a
            x = c - slopes[h] * dist if slopes is not None else c
            e = torch.where(see[b], torch.exp(x), torch.zeros_like(x))
            p = e / (1 + e.sum(1, keepdim=True))
            o[b, :, h] = p @ vv[b, :, h]
            to[b, :, h] = p @ vv[b, :, h].abs()
            if do is None:
                continue
            g = do[b, :, h]
            g = torch.where(sees[b, :, None], g, torch.zeros_like(g))
            dp = g @ vv[b, :, h].T
            D = (p * dp).sum(1, keepdim=True)
            Dabs = (g.abs() * o[b, :, h].abs()).sum(1, keepdim=True)
            w = rw * (1 - (c / cap) ** 2) if cap else torch.full_like(c, rw)
            ds = -p * (dp - D) * w
            dsabs = p * ((g.abs() @ vv[b, :, h].abs().T) + 2 * Dabs) * w
            sg = torch.sign(d)
            dq[b, :, h] = (ds[:, :, None] * sg).sum(1)
            tq[b, :, h] = dsabs.sum(1)[:, None]
            dkk[b, :, h] = -(ds[:, :, None] * sg).sum(0)
            tkk[b, :, h] = dsabs.sum(0)[:, None]
            dvv[b, :, h] = p.T @ g
            tvv[b, :, h] = p.T @ g.abs()
    if do is None:
        return [o], [to]
    f = lambda x: x.unflatten(2, (Hk, G)).sum(3)  # noqa: E731
    return [o, dq, f(dkk), f(dvv)], [to, tq, f(tkk), f(tvv)]


def check(got, ref, terms, dtype, W, names=("o", "dq", "dk", "dv")):
    u = torch.finfo(dtype).eps / 2
    F = 2.0 ** -24 * (3 * W + 64)
    for x, r, t, n in zip(got, ref, terms, names):
        x = x.detach().double().cpu()
        assert x.shape == r.shape and torch.isfinite(x).all(), n
        more = t * F + (t * u if dtype != torch.float32 else 0)
        # values below the type's normal numbers are off by half of its smallest step
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        over = (x - r).abs() - (u * r.abs() + more + tiny)
        assert (over <= 0).all(), "%s: off by %.3g where %.3g is allowed" % (
            n, (x - r).abs().flatten()[over.argmax()], ((x - r).abs() - over).flatten()[over.argmax()])
