"""Plain statements in 64 bits of the masked attention and of the paged 8-bit cache, with what rounding may do to them.

masked() returns o, dq, dk, dv and, for each, the sum of the magnitudes of its terms: a result computed in float32 from inputs
of a type whose half step is u = finfo.eps / 2, and rounded once to that type, is off by at most

    u * |result| + u * terms + F * terms

The first part is the output's rounding.  The second is there for 16-bit inputs: a logit from 16-bit codes is off by up to u (6.5
times its rms, at the widest range that codes are taken for), which is a relative error u of a term.  F = 2^-24 * (3 W + 64):
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


class PlainCache:
    """The paged cache, one token and one page at a time, on the host."""

    def __init__(self, N, P, Hk, W, Wv, rows, M):
        self.N, self.P, self.Hk, self.W, self.Wv, self.rows, self.M = N, P, Hk, W, Wv, rows, M
        r16 = lambda w: -(-w // 16) * 16  # noqa: E731
        self.pages = [torch.zeros(N, Hk, P, r16(w), dtype=torch.int8) for w in (W, Wv)]
        self.scale = [torch.zeros(N, Hk) for _ in range(2)]
        self.table = torch.full((rows, M), -1, dtype=torch.int32)
        self.lens, self.refs = [0] * rows, [0] * N
        self.stack = list(range(N - 1, -1, -1))

    def _once(self, seqs):
        seen = set()
        for b, s in enumerate(seqs):
            ok = 0 <= s < self.rows and s not in seen
            seen.add(s)
            yield b, s, ok

    def append(self, k, v, seqs=None, counts=None):
        B, n = k.shape[:2]
        P = self.P
        seqs = list(range(B)) if seqs is None else seqs
        counts = [n] * B if counts is None else [min(max(c, 0), n) for c in counts]
        served = [False] * B
        refs0 = list(self.refs)
        left = []
        empty = False
        jobs = []
        for b, s, ok in self._once(seqs):
            start, cnt = (self.lens[s], counts[b]) if ok else (0, 0)
            if not ok or start + cnt > self.M * P:
                continue
            last = int(self.table[s, start // P]) if start % P and cnt else -1
            if start % P and cnt and not 0 <= last < self.N:
                continue
            share = last >= 0 and refs0[last] > 1
            need = (-(-(start + cnt) // P) - -(-start // P) if cnt else 0) + share
            if need and (empty or need > len(self.stack)):
                empty = True
                continue
            served[b] = True
            got = []
            for j in range(start // P, -(-(start + cnt) // P) if cnt else 0):
                if j * P < start and not share:
                    got.append((last, last))
                else:
                    page = self.stack.pop()
                    self.refs[page] = 1
                    got.append((page, last if j * P < start else -1))
                self.table[s, j] = got[-1][0]
            if share:
                left.append(last)
            jobs.append((b, s, start, cnt, got))
        for b, s, start, cnt, got in jobs:
            for (page, src), j in zip(got, range(start // P, self.M)):
                for side, x in enumerate((k, v)):
                    self._write(side, page, src, j, start, cnt, x[b].float())
            self.lens[s] = start + cnt
        gone = []
        for p in left:
            self.refs[p] -= 1
            if self.refs[p] == 0:
                gone.append(p)
        self.stack += sorted(gone)
        return served

    def _write(self, side, page, src, j, start, cnt, x):
        P, w = self.P, (self.W, self.Wv)[side]
        lo, hi = max(start, j * P), min(start + cnt, (j + 1) * P)
        new = x[lo - start:hi - start]  # [m, Hk, w]
        mag = torch.where(torch.isfinite(new), new.abs(), torch.zeros_like(new))
        now = mag.amax((0, 2)) * (1.0 / 127.0)
        had = max(0, start - j * P)
        if had:
            held = self.scale[side][src]
            now = torch.maximum(held, now)
            ratio = torch.where(now > 0, held / now, torch.zeros_like(now))
            codes = self.pages[side][src, :, :had].float()
            self.pages[side][page, :, :had] = torch.round(codes * ratio[:, None, None]).to(torch.int8)
        div = torch.where(now > 0, now, torch.ones_like(now))
        c = torch.round(new / div[None, :, None]).clamp(-127, 127)
        c = torch.where(torch.isnan(new), torch.zeros_like(c), c)
        self.pages[side][page, :, lo - j * P:hi - j * P, :w] = c.transpose(0, 1).to(torch.int8)
        self.pages[side][page, :, lo - j * P:hi - j * P, w:] = 0
        self.scale[side][page] = now

    def fork(self, parents, children):
        lens0, rows0 = list(self.lens), self.table.clone()
        served = []
        for b, c, ok in self._once(children):
            p = parents[b]
            ok = ok and 0 <= p < self.rows and p != c and lens0[c] == 0
            served.append(ok)
            if ok:
                for j in range(-(-lens0[p] // self.P)):
                    self.table[c, j] = rows0[p, j]
                    self.refs[int(rows0[p, j])] += 1
                self.lens[c] = lens0[p]
        return served

    def free(self, seqs, keep=None):
        gone = []
        for b, s, ok in self._once(seqs):
            if not ok:
                continue
            kept = 0 if keep is None else min(max(keep[b], 0), self.lens[s])
            for j in range(-(-kept // self.P), -(-self.lens[s] // self.P)):
                p = int(self.table[s, j])
                self.table[s, j] = -1
                self.refs[p] -= 1
                if self.refs[p] == 0:
                    gone.append(p)
            self.lens[s] = kept
        self.stack += sorted(gone)

    def compact(self):
        live = [p for p in range(self.N) if self.refs[p]]
        n = len(live)
        holes = [p for p in range(n) if not self.refs[p]]
        for to, p in zip(holes, [p for p in live if p >= n]):
            for x in self.pages + self.scale:
                x[to] = x[p]
            self.refs[to], self.refs[p] = self.refs[p], 0
            self.table[self.table == p] = to
        self.stack = list(range(self.N - 1, n - 1, -1))
        return n

    def tokens(self, s):
        """Keys and values of a sequence in 64 bits, [len, Hk, w]."""
        pages = self.table[s, :-(-self.lens[s] // self.P)].long()
        return [(self.pages[x][pages].double() * self.scale[x][pages].double()[:, :, None, None]).transpose(1, 2).flatten(0, 1)[:self.lens[s], :, :w]
                for x, w in ((0, self.W), (1, self.Wv))]

    def attend(self, q, seqs=None, counts=None, cap=0.0, slopes=None):
        B, n, H, W = q.shape
        q = q.double().cpu()
        out, terms = torch.zeros(B, n, H, self.Wv, dtype=torch.float64), torch.zeros(B, n, H, self.Wv, dtype=torch.float64)
        for b in range(B):
            s = b if seqs is None else seqs[b]
            if not 0 <= s < self.rows or not self.lens[s]:
                continue
            k, v = self.tokens(s)
            cnt = n if counts is None else min(max(counts[b], 0), n)
            for t in range(cnt):
                m = self.lens[s] - cnt + t + 1
                if m < 1:
                    continue
                for h in range(H):
                    hk = h // (H // self.Hk)
                    x = -(q[b, t, h] - k[:m, hk]).abs().sum(1) / math.sqrt(W)
                    x = cap * torch.tanh(x / cap) if cap else x
                    x = x - (slopes[h] * torch.arange(m - 1, -1, -1).double() if slopes is not None else 0.0)
                    p = torch.exp(x)
                    p = p / (1 + p.sum())
                    out[b, t, h], terms[b, t, h] = p @ v[:m, hk], p @ v[:m, hk].abs()
        return out, terms
