"""The masked L1 attention, its backward, and the paged 8-bit cache that serves it: what is measured of them.

Masked attention (training and prefill).  q [B,T,H,W], k [B,S,Hk,W], v [B,S,Hk,Wv], T <= S, H a multiple of Hk, query head h reads
key head h // (H/Hk); query t is token i = S-T+t of its row of the batch.

    a[t,s] = -1/sqrt(W) * sum_w |q[t,w] - k[s,w]|          c = cap * tanh(a / cap)   (cap > 0; else c = a)
    x[t,s] = c - slope[h] * |i - s|                         p[t,s] = exp(x) / (1 + sum_s exp(x)) over the visible s
    o[t]   = sum_s p[t,s] * v[s]

s is visible to i where (not causal, or s <= i, or s < prefix[b]) and, with documents, doc[b,s] == doc[b,i] >= 0.
A row that sees nothing is zero.

Paged cache.  A page holds `page` tokens of every key head as 8-bit codes, one scale for each page and head:
value = code * scale.  append() writes new tokens (a page whose largest magnitude grows is coded again), attend() is the attention
above for the last tokens of each sequence, causal, over the cache; fork() shares a sequence's pages with a new one, free() gives
pages back (all, or those behind a kept length), compact() moves the pages in use to the front of the pool.

own = False computes all of it with elementary torch operations; own = True calls the framework."""
import math
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


# ------------------------------------------------------------------------------------------------------------------ cases

def listed():
    m = dict(op="masked", Wv=0, causal=True, docs=0, prefix=False, cap=0.0, slopes=False, backward=True)
    return [
        # one short sequence of a small model, answered by itself: only latency counts
        dict(m, name="masked_fwd_short", B=1, T=64, S=64, H=8, Hk=8, W=32, dtype="bf16", backward=False),
        # the second half of a prompt against all of it, grouped heads, distance bias (prefill in chunks)
        dict(m, name="masked_fwd_chunk", B=2, T=1024, S=2048, H=16, Hk=4, W=64, dtype="bf16", backward=False, slopes=True),
        # a training step in float32 on packed documents, the type that the dense operator trains in
        dict(m, name="masked_train_f32_docs", B=4, T=1024, S=1024, H=8, Hk=8, W=64, dtype="f32", docs=7),
        # a training step on odd sizes: a prefix that sees itself, capped scores, shared key heads, widths that pad
        dict(m, name="masked_train_f16_prefix", B=3, T=777, S=777, H=8, Hk=2, W=96, Wv=65, dtype="f16", prefix=True, cap=6.0, slopes=True),
        # the largest: one long sequence of packed documents and one of the heads' ordinary width
        dict(m, name="masked_train_bf16_long", B=1, T=4096, S=4096, H=16, Hk=16, W=64, dtype="bf16", docs=3),
        # one user's next token after a short conversation: latency
        dict(op="paged", name="attend_one", B=1, n=1, least=300, most=300, H=8, Hk=8, W=64, Wv=64, page=16, cap=0.0, slopes=False, dtype="bf16"),
        # a batch of conversations of uneven lengths, grouped heads, distance bias
        dict(op="paged", name="attend_batch", B=32, n=1, least=100, most=4000, H=16, Hk=4, W=64, Wv=64, page=32, cap=0.0, slopes=True, dtype="bf16"),
        # long documents, four drafted tokens each, wide heads, capped scores
        dict(op="paged", name="attend_long_draft", B=16, n=4, least=8192, most=32768, H=16, Hk=4, W=128, Wv=128, page=64, cap=20.0, slopes=False, dtype="f16"),
        # the token that each sequence of a batch gets in a decode step, drafted and rejected: append and give back
        dict(op="append", name="append_step", B=64, n=1, least=40, most=2000, Hk=4, W=64, Wv=64, page=32, dtype="bf16"),
        # prompts that come in: many full pages in each row, ragged
        dict(op="append", name="append_prompts", B=8, n=2000, least=0, most=100, Hk=8, W=128, Wv=128, page=64, dtype="bf16"),
        # beam search: every parent forked, the children go on for a few tokens and are dropped
        dict(op="fork", name="fork_beams", B=64, ways=4, n=3, least=500, most=4000, Hk=4, W=64, Wv=64, page=32, dtype="bf16"),
        # a pool with holes, its pages moved to the front so that the rest can be handed back
        dict(op="compact", name="compact_pool", B=128, least=200, most=6000, Hk=4, W=64, Wv=64, page=32, dtype="bf16"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(("masked", "masked", "masked", "paged", "paged", "append", "fork", "compact"))
    Hk = rng.choice((1, 2, 4, 8))
    W, Wv = rng.choice((32, 33, 64, 64, 65, 96, 128)), rng.choice((32, 64, 64, 96, 128))
    if op == "masked":
        H = Hk * rng.choice((1, 2, 4))
        S = _log(rng, 1, 2500)
        T = S if rng.random() < 0.6 else rng.randint(1, S)
        T = max(1, min(T, int(1.2e8 // (S * H))))
        B = max(1, min(rng.randint(1, 6), int(6e7 // (T * S * H))))
        return dict(op=op, B=B, T=T, S=S, H=H, Hk=Hk, W=W, Wv=rng.choice((0, Wv)), dtype=rng.choice(("f32", "f16", "bf16")), causal=rng.random() < 0.8,
                    docs=rng.choice((0, 0, 2, 5)), prefix=rng.random() < 0.3, cap=rng.choice((0.0, 0.0, 4.0, 30.0)), slopes=rng.random() < 0.4,
                    backward=rng.random() < 0.6)
    page = rng.choice((16, 32, 64))
    most = _log(rng, 20, 8000)
    c = dict(op=op, B=_log(rng, 1, 64), least=rng.randint(0, most), most=most, Hk=Hk, W=rng.choice((32, 64, 96, 128)), Wv=rng.choice((32, 64, 96, 128)), page=page,
             dtype=rng.choice(("f16", "bf16", "f32")))
    if op == "paged":
        c.update(n=rng.choice((1, 1, 1, 2, 5)), H=Hk * rng.choice((1, 2, 4, 8)), cap=rng.choice((0.0, 8.0)), slopes=rng.random() < 0.5)
        c["B"] = max(1, min(c["B"], int(8e6 // (most * c["H"])), int(2e7 // (most * c["H"] * c["n"])), int(1.2e6 // (most * Hk))))
    if op == "append":
        c.update(n=_log(rng, 1, 1500))
        c["B"] = max(1, min(c["B"], 120000 // (c["n"] * Hk), int(1.2e6 // (most * Hk))))
    if op == "fork":
        c.update(ways=rng.randint(1, 5), n=rng.randint(1, 40))
        c["B"] = max(1, min(c["B"], int(1.2e6 // (most * Hk))))
    if op == "compact":
        c["B"] = max(1, min(c["B"], int(1.2e6 // (most * Hk))))
    return c


# ----------------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    return (_prepare_masked if case["op"] == "masked" else _prepare_paged)(case, g)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE).to(DTYPES[dtype])


def _slopes(c):
    return tuple(2.0 ** (-8.0 * (h + 1) / c["H"]) for h in range(c["H"])) if c["slopes"] else None


def _prepare_masked(c, g):
    B, T, S, H, Hk, W = (c[k] for k in ("B", "T", "S", "H", "Hk", "W"))
    Wv = c["Wv"] or W
    s = dict(case=c, slopes=_slopes(c), doc=None, prefix=None)
    s["q"], s["k"], s["v"] = _randn(g, c["dtype"], B, T, H, W), _randn(g, c["dtype"], B, S, Hk, W), _randn(g, c["dtype"], B, S, Hk, Wv)
    if c["docs"]:  # documents of uneven lengths one after the other, padding (-1) behind the last of them
        cuts = torch.randint(0, S + 1, (B, c["docs"]), generator=g, device=DEVICE, dtype=torch.int32).sort(1).values
        at = torch.arange(S, device=DEVICE, dtype=torch.int32)
        doc = (at[None, :, None] >= cuts[:, None, :]).sum(2, dtype=torch.int32)
        s["doc"] = torch.where(at[None] < S - (S // 50), doc, torch.full_like(doc, -1))
    if c["prefix"]:
        s["prefix"] = torch.randint(0, S // 2 + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
    if c["backward"]:
        s["do"] = _randn(g, c["dtype"], B, T, H, Wv)
        for n in "qkv":
            s[n].requires_grad_()
    return s


def _prepare_paged(c, g):
    B, Hk, W, Wv, P, op = (c[k] for k in ("B", "Hk", "W", "Wv", "page", "op"))
    n = c.get("n", 0)
    rows = B * (1 + c.get("ways", 0))  # table rows: the children of a fork start empty
    ways = c.get("ways", 0)
    lens = torch.randint(c["least"], c["most"] + 1, (B,), generator=g, device=DEVICE)
    if op == "paged":
        lens = lens.clamp_min(n)
    used = (lens + P - 1) // P
    M = (c["most"] + n + P - 1) // P + 1  # pages that a row of the table holds
    more = ((n + P - 1) // P + 1) * B * max(1, ways) if n and op != "paged" else 0
    N = B * ((max(c["most"], n) + P - 1) // P) + more + 3
    if op == "compact":
        N = 2 * N
    perm = torch.randperm(N, generator=g, device=DEVICE).to(torch.int32)  # where a page lies in the pool says nothing
    first = torch.cumsum(used, 0) - used
    j = torch.arange(M, device=DEVICE)
    table = torch.full((rows, M), -1, dtype=torch.int32, device=DEVICE)
    table[:B] = torch.where(j[None] < used[:, None], perm[(first[:, None] + j[None]).clamp_max(N - 1)], -1)
    refs = torch.zeros(N, dtype=torch.int32, device=DEVICE)
    n_used = int(used.sum())
    refs[perm[:n_used].long()] = 1
    free = torch.zeros(N, dtype=torch.int32, device=DEVICE)
    free[:N - n_used] = perm[n_used:]
    all_lens = torch.zeros(rows, dtype=torch.int32, device=DEVICE)
    all_lens[:B] = lens.to(torch.int32)
    pool = dict(k_pages=torch.randint(-127, 128, (N, Hk, P, W), generator=g, device=DEVICE, dtype=torch.int8),
                v_pages=torch.randint(-127, 128, (N, Hk, P, Wv), generator=g, device=DEVICE, dtype=torch.int8),
                k_scale=(torch.rand(N, Hk, generator=g, device=DEVICE) + 2.0) / 127, v_scale=(torch.rand(N, Hk, generator=g, device=DEVICE) + 2.0) / 127,
                table=table, lens=all_lens, refs=refs, free=free, n_free=torch.tensor([N - n_used], dtype=torch.int32, device=DEVICE))
    s = dict(case=c, pool=pool)
    if op == "paged":
        s.update(q=_randn(g, c["dtype"], B, n, c["H"], W), slopes=_slopes(c))
    if op == "append":
        s.update(k=_randn(g, c["dtype"], B, n, Hk, W), v=_randn(g, c["dtype"], B, n, Hk, Wv), back=all_lens.clone(),
                 seqs=torch.arange(B, dtype=torch.int32, device=DEVICE),
                 counts=torch.randint((n + 1) // 2, n + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32))
    if op == "fork":
        s["parents"] = torch.arange(B, dtype=torch.int32, device=DEVICE).repeat_interleave(ways)
        s["children"] = torch.arange(B, rows, dtype=torch.int32, device=DEVICE)
        s.update(k=_randn(g, c["dtype"], B * ways, n, Hk, W), v=_randn(g, c["dtype"], B * ways, n, Hk, Wv))
    if op == "compact":
        s["kept"] = {k: pool[k].clone() for k in ("table", "refs", "free", "n_free")}
    return s


# -------------------------------------------------------------------------------------------------------------------- run

def _framework():
    if "l1-attention_amd" not in sys.path:
        sys.path.insert(1, "l1-attention_amd")
    import l1attn_masked_cuda
    import l1attn_paged_cuda
    return l1attn_masked_cuda, l1attn_paged_cuda


def run(s):
    return {"masked": _run_masked, "paged": _run_attend, "append": _run_append, "fork": _run_fork, "compact": _run_compact}[s["case"]["op"]](s)


def _run_masked(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            return plain_masked(s["q"], s["k"], s["v"], s["doc"], s["prefix"], c["causal"], c["cap"], s["slopes"], s.get("do"))
    if "op" not in s:  # the module is a part of the model
        s["op"] = _framework()[0].L1AttnMasked(causal=c["causal"], softcap=c["cap"], slopes=s["slopes"])
    if not c["backward"]:
        with torch.no_grad():
            return [s["op"](s["q"], s["k"], s["v"], doc=s["doc"], prefix=s["prefix"])]
    o = s["op"](s["q"], s["k"], s["v"], doc=s["doc"], prefix=s["prefix"])
    return [o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])]


def _cache(s):
    if "cache" not in s:  # the handle that a server keeps
        s["cache"] = _framework()[1].L1PagedCache(**s["pool"])
    return s["cache"]


def _run_attend(s):
    c = s["case"]
    if own:
        return [_framework()[1].l1attn_paged(s["q"], _cache(s), softcap=c["cap"], slopes=s["slopes"])]
    return [plain_attend(s["q"], s["pool"], c["cap"], s["slopes"])]


STATE = ("table", "lens", "refs", "free", "n_free")
CODES = ("k_pages", "v_pages", "k_scale", "v_scale")  # the cache as it is held: codes, which have to be equal, and the scales that give them their values


def _run_append(s):
    if own:
        served = _cache(s).append(s["k"], s["v"], seqs=s["seqs"], counts=s["counts"])
        grown = s["pool"]["lens"].clone()
        _cache(s).free(s["seqs"], keep=s["back"])
    else:
        served = plain_append(s["pool"], s["k"], s["v"], s["seqs"], s["counts"])
        grown = s["pool"]["lens"].clone()
        plain_free(s["pool"], s["seqs"], s["back"])
    return [served, grown] + [s["pool"][n] for n in STATE + CODES]


def _run_fork(s):
    if own:
        forked = _cache(s).fork(s["parents"], s["children"])
        served = _cache(s).append(s["k"], s["v"], seqs=s["children"])
        grown = s["pool"]["table"].clone()
        _cache(s).free(s["children"])
    else:
        forked = plain_fork(s["pool"], s["parents"], s["children"])
        served = plain_append(s["pool"], s["k"], s["v"], s["children"], None)
        grown = s["pool"]["table"].clone()
        plain_free(s["pool"], s["children"], None)
    return [forked, served, grown] + [s["pool"][n] for n in STATE + CODES]


def _run_compact(s):
    for n, t in s["kept"].items():  # the holes are there again: the pages that move lie where they lay
        s["pool"][n].copy_(t)
    live = _cache(s).compact() if own else plain_compact(s["pool"])
    return [live] + [s["pool"][n] for n in STATE + CODES]


# ------------------------------------------------------------------------------------------------------------ plain forms

def _scores(q, k, i, s, cap, slopes):
    """The differences q - k [B,t,s,H,W], the capped score c and the logit x [B,t,s,H] of the queries at places i."""
    d = q[:, :, None] - k[:, None]
    c = d.abs().sum(-1) * (-1.0 / math.sqrt(q.shape[-1]))
    if cap:
        c = cap * torch.tanh(c / cap)
    x = c
    if slopes is not None:
        x = c - torch.tensor(slopes, device=q.device, dtype=torch.float32) * (i[:, None] - s[None]).abs()[..., None]
    return d, c, x


def plain_masked(q, k, v, doc, prefix, causal, cap, slopes, do):
    B, T, H, W = q.shape
    S, Hk, Wv, G, dt = k.shape[1], k.shape[2], v.shape[3], H // k.shape[2], q.dtype
    kf, vf = (x.float().repeat_interleave(G, 2) for x in (k, v))
    at = torch.arange(S, device=q.device)
    o = torch.empty(B, T, H, Wv, device=q.device)
    if do is not None:
        dq = torch.empty(B, T, H, W, device=q.device)
        dk, dv = torch.zeros(B, S, H, W, device=q.device), torch.zeros(B, S, H, Wv, device=q.device)
    step = max(1, int(5e8 // (B * S * H * W)))
    for t in range(0, T, step):  # rows of queries at a time: the differences of all of them do not fit
        r = slice(t, min(T, t + step))
        i = at[S - T:][r]
        see = torch.ones(B, i.numel(), S, dtype=torch.bool, device=q.device)
        if causal:
            see &= at[None] <= i[:, None]
            if prefix is not None:
                see |= at[None, None] < prefix[:, None, None]
        if doc is not None:
            see &= (doc[:, i, None] == doc[:, None]) & (doc[:, i, None] >= 0)
        d, c, x = _scores(q[:, r].float(), kf, i, at, cap, slopes)
        e = torch.exp(x) * see[..., None]
        p = e / (1.0 + e.sum(2, keepdim=True))
        ph = p.permute(0, 3, 1, 2)
        o[:, r] = (ph @ vf.permute(0, 2, 1, 3)).permute(0, 2, 1, 3)
        if do is None:
            continue
        dof = do[:, r].float()
        dp = (dof.permute(0, 2, 1, 3) @ vf.permute(0, 2, 3, 1)).permute(0, 2, 3, 1)
        ds = p * (dp - (p * dp).sum(2, keepdim=True))
        if cap:
            ds = ds * (1.0 - (c / cap) ** 2)
        sg = torch.sign(d).mul_((ds * (-1.0 / math.sqrt(W)))[..., None])
        dq[:, r] = sg.sum(2)
        dk -= sg.sum(1)
        dv += (ph.transpose(2, 3) @ dof.permute(0, 2, 1, 3)).permute(0, 2, 1, 3)
    if do is None:
        return [o.to(dt)]
    return [o.to(dt), dq.to(dt), dk.unflatten(2, (Hk, G)).sum(3).to(dt), dv.unflatten(2, (Hk, G)).sum(3).to(dt)]


def _gather(pages, scale, table, M):
    """The tokens of each sequence in order, [B, M*page, Hk, W] in float32; pages that are not there give zeros."""
    at = table.clamp_min(0).long()
    x = pages[at].float() * scale[at][..., None, None]  # [B,M,Hk,P,W]
    return x.permute(0, 1, 3, 2, 4).flatten(1, 2)


def plain_attend(q, pool, cap, slopes):
    B, n, H, W = q.shape
    P, Hk = pool["k_pages"].shape[2], pool["k_pages"].shape[1]
    table, lens = pool["table"][:B], pool["lens"][:B].long()
    k, v = (_gather(pool[a + "_pages"], pool[a + "_scale"], table, table.shape[1]) for a in "kv")
    S, G = k.shape[1], H // Hk
    at = torch.arange(S, device=q.device)
    i = lens[:, None] - n + torch.arange(n, device=q.device)  # [B,n]
    qf = q.float().unflatten(2, (Hk, G))  # [B,n,Hk,G,W]
    a = torch.empty(B, n, Hk, G, S, device=q.device)
    for t in range(n):
        a[:, t] = (qf[:, t, :, :, None] - k.permute(0, 2, 1, 3)[:, :, None]).abs_().sum(-1)
    x = a.mul_(-1.0 / math.sqrt(W))
    if cap:
        x = cap * torch.tanh(x / cap)
    if slopes is not None:
        x = x - torch.tensor(slopes, device=q.device, dtype=torch.float32).view(1, 1, Hk, G, 1) * (i[:, :, None] - at).abs()[:, :, None, None]
    e = torch.exp(x) * (at[None, None] <= i[:, :, None])[:, :, None, None]
    e = e / (1.0 + e.sum(-1, keepdim=True))
    o = e.permute(0, 2, 1, 3, 4).flatten(2, 3) @ v.permute(0, 2, 1, 3)  # [B,Hk,n*G,Wv]
    return o.unflatten(2, (n, G)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(q.dtype)


def plain_append(pool, k, v, seqs, counts):
    B, n = k.shape[:2]
    P, M, N = pool["k_pages"].shape[2], pool["table"].shape[1], pool["refs"].shape[0]
    dev = k.device
    seqs = seqs.long()
    start = pool["lens"][seqs].long()
    cnt = torch.full((B,), n, device=dev) if counts is None else counts.long().clamp(0, n)
    rows = pool["table"][seqs].long()
    last = rows.gather(1, (start // P).clamp_max(M - 1)[:, None])[:, 0]
    share = (start % P > 0) & (cnt > 0) & (pool["refs"][last.clamp_min(0)] > 1)  # a shared page that is written to: a copy of its own
    fresh = (start + cnt + P - 1) // P - (start + P - 1) // P
    fits = start + cnt <= M * P
    need = (fresh + share) * fits
    upto = torch.cumsum(need, 0)
    n_free = pool["n_free"].long()
    served = ((upto <= n_free) | (need == 0)) & fits  # once the pool is empty, no later row that needs a page is served
    need, cnt, share = need * served, cnt * served, share & served
    J = (n + P - 1) // P + 1
    j = torch.arange(J, device=dev)
    base = start // P
    touched = (j[None] < ((start + cnt + P - 1) // P - base)[:, None]) & (cnt > 0)[:, None]
    took = (upto - need)[:, None] + j[None] - ((start % P > 0) & ~share).long()[:, None]
    is_new = touched & ((j[None] > 0) | (start % P == 0)[:, None] | share[:, None])
    place = (base[:, None] + j[None]).clamp_max(M - 1)
    old = rows.gather(1, place)
    got = pool["free"].long()[(n_free - 1 - took).clamp(0, N - 1)]
    dst = torch.where(is_new, got, old)
    flat = (seqs[:, None] * M + base[:, None] + j[None])[touched]
    pool["table"].view(-1)[flat] = dst[touched].to(torch.int32)
    # pages: codes of the tokens that were there, then those of the new ones, with one scale
    token = (base[:, None, None] + j[None, :, None]) * P + torch.arange(P, device=dev)  # [B,J,P]
    new = (token >= start[:, None, None]) & (token < (start + cnt)[:, None, None])
    was = token < start[:, None, None]
    src = (token - start[:, None, None]).clamp(0, n - 1)
    b = torch.arange(B, device=dev)[:, None, None]
    at = touched.nonzero(as_tuple=True)
    for pages, scale, x in (("k_pages", "k_scale", k), ("v_pages", "v_scale", v)):
        y = x[b.expand_as(src)[at], src[at]].float().transpose(1, 2)  # [touched, Hk, P, W]
        isn, isw = new[at][:, None, :, None], was[at][:, None, :, None]
        codes = pool[pages][old.clamp_min(0)[at]].float()
        held = pool[scale][old.clamp_min(0)[at]] * isw.any(2)[..., 0]
        now = torch.maximum(held, (y.abs() * isn).amax((2, 3)) / 127.0)
        ratio = torch.where(now > 0, held / now, torch.zeros_like(now))
        div = torch.where(now > 0, now, torch.ones_like(now))
        again = torch.round(codes * ratio[..., None, None])
        coded = torch.round(y / div[..., None, None]).clamp(-127, 127)
        there = pool[pages][dst[at]].float()
        pool[pages][dst[at]] = torch.where(isn, coded, torch.where(isw, again, there)).to(torch.int8)
        pool[scale][dst[at]] = now
    # references: new pages have one, the shared ones that were copied lose one
    pool["refs"].index_put_((dst[is_new],), torch.ones((), dtype=torch.int32, device=dev))
    before = pool["refs"].clone()
    pool["refs"].index_add_(0, last.clamp_min(0), -share.to(torch.int32))
    pool["n_free"] -= need.sum().to(torch.int32)
    pool["lens"][seqs] = (start + cnt).to(torch.int32)
    _push(pool, (pool["refs"] == 0) & (before > 0))
    return served


def _push(pool, freed):
    """Pages that are no longer used go on top of the free ones, in ascending order."""
    N = freed.shape[0]
    at = pool["n_free"] + torch.cumsum(freed, 0) - 1
    room = torch.cat([pool["free"], pool["free"][:1]])
    room[torch.where(freed, at, N)] = torch.arange(N, dtype=torch.int32, device=freed.device)
    pool["free"].copy_(room[:N])
    pool["n_free"] += freed.sum().to(torch.int32)


def plain_free(pool, seqs, keep):
    P, M = pool["k_pages"].shape[2], pool["table"].shape[1]
    seqs = seqs.long()
    lens = pool["lens"][seqs]
    keep = torch.zeros_like(lens) if keep is None else torch.minimum(keep, lens).clamp_min(0)
    j = torch.arange(M, device=lens.device)[None]
    rows = pool["table"][seqs]
    drop = (j >= ((keep + P - 1) // P)[:, None]) & (j < ((lens + P - 1) // P)[:, None]) & (rows >= 0)
    before = pool["refs"].clone()
    pool["refs"].index_add_(0, rows.clamp_min(0).view(-1).long(), -drop.view(-1).to(torch.int32))
    pool["table"][seqs] = torch.where(drop, -1, rows)
    pool["lens"][seqs] = keep
    _push(pool, (pool["refs"] == 0) & (before > 0))


def plain_fork(pool, parents, children):
    parents, children = parents.long(), children.long()
    P = pool["k_pages"].shape[2]
    served = (pool["lens"][children] == 0) & (parents != children)
    lens = pool["lens"][parents]
    rows = pool["table"][parents]
    j = torch.arange(rows.shape[1], device=rows.device)[None]
    takes = (j < ((lens + P - 1) // P)[:, None]) & served[:, None] & (rows >= 0)
    pool["refs"].index_add_(0, rows.clamp_min(0).view(-1).long(), takes.view(-1).to(torch.int32))
    pool["table"][children] = torch.where(takes, rows, pool["table"][children])
    pool["lens"][children] = torch.where(served, lens, pool["lens"][children])
    return served


def plain_compact(pool):
    N = pool["refs"].shape[0]
    dev = pool["refs"].device
    live = pool["refs"] > 0
    n_live = live.sum()
    at = torch.arange(N, device=dev)
    holes, movers = (~live & (at < n_live)).nonzero()[:, 0], (live & (at >= n_live)).nonzero()[:, 0]
    for n in ("k_pages", "v_pages", "k_scale", "v_scale", "refs"):
        pool[n][holes] = pool[n][movers]
    pool["refs"][movers] = 0
    to = at.to(torch.int32)
    to[movers] = holes.to(torch.int32)
    pool["table"].copy_(torch.where(pool["table"] >= 0, to[pool["table"].clamp_min(0).long()], -1))
    left = N - n_live
    pool["free"].copy_(torch.where(at < left, N - 1 - at, pool["free"].long()).to(torch.int32))
    pool["n_free"].copy_(left.view(1).to(torch.int32))
    return n_live.view(1).to(torch.int32)


# ------------------------------------------------------------------------------------------------------------------- work

def _pairs(c):
    """Visible (query, key) pairs of one head and row, with documents at their expected share."""
    T, S = c["T"], c["S"]
    n = T * S - T * (T - 1) / 2 if c["causal"] else T * S
    if c["causal"] and c["prefix"]:
        n += (S // 4) ** 2 / 2
    return n * (2.0 / (c["docs"] + 2) if c["docs"] else 1.0)


def work(c):
    b = {"f32": 4, "f16": 2, "bf16": 2}[c["dtype"]]
    if c["op"] == "masked":
        Wv = c["Wv"] or c["W"]
        qo, kv = c["B"] * c["T"] * c["H"] * (c["W"] + Wv) * b, c["B"] * c["S"] * c["Hk"] * (c["W"] + Wv) * b
        n = _pairs(c) * c["B"] * c["H"]
        if not c["backward"]:
            return {"bytes": qo + kv, "flops": n * (2 * c["W"] + 2 * Wv)}
        # forward: difference, sum, value product; backward: the scores again, two value products, sign and two sums
        return {"bytes": 2 * (qo + kv) + c["B"] * c["T"] * c["H"] * Wv * b, "flops": n * (2 * c["W"] + 2 * Wv + 2 * c["W"] + 4 * Wv + 4 * c["W"])}
    mean = (c["least"] + c["most"]) / 2
    token = c["Hk"] * (c["W"] + c["Wv"])
    if c["op"] == "paged":
        return {"bytes": c["B"] * (mean * token + c["n"] * c["H"] * (c["W"] + c["Wv"]) * b), "flops": c["B"] * mean * c["n"] * c["H"] * 2 * (c["W"] + c["Wv"])}
    if c["op"] == "append":
        tokens = c["B"] * (c["n"] + (c["n"] + 1) // 2) / 2
        return {"bytes": tokens * token * (b + 1), "flops": tokens * token * 3}
    if c["op"] == "fork":
        tokens = c["B"] * c["ways"] * c["n"]
        return {"bytes": tokens * token * (b + 1) + c["B"] * c["ways"] * (c["page"] * token + 8 * mean / c["page"]), "flops": tokens * token * 3}
    # half of the pool is free, so half of the pages in use lie behind the place that they move to
    return {"bytes": c["B"] * mean * token, "flops": 0}


# ------------------------------------------------------------------------------------------------------------------ exact

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "masked":
        return _exact_masked(s)
    if case["op"] == "paged":
        return _exact_attend(s)
    if case["op"] == "append":
        # the scales of a page are those of its values; what the codes are stands in whole numbers beside them
        k_scale, v_scale = (_exact_scales(s, n) for n in "kv")
        return [None] * 9 + [k_scale, v_scale]
    if case["op"] == "fork":
        return [None] * 10 + [_exact_fork_scales(s, n) for n in "kv"]
    refs = s["pool"]["refs"].tolist()
    used = [p for p, r in enumerate(refs) if r > 0]
    into = dict(zip([p for p in range(len(used)) if refs[p] == 0], [p for p in used if p >= len(used)]))
    moved = torch.tensor([into.get(p, p) for p in range(len(refs))], device=s["pool"]["refs"].device)
    return [None] * 8 + [s["pool"][n + "_scale"].double()[moved] for n in "kv"]


def _exact_masked(s):
    c = s["case"]
    B, T, S, H, Hk = (c[n] for n in ("B", "T", "S", "H", "Hk"))
    if _pairs(dict(c, causal=False, docs=0)) * B * H * c["W"] > 3e10:
        return None
    q, k, v = (s[n].detach().double() for n in "qkv")
    out = [torch.zeros(B, T, H, v.shape[3], dtype=torch.float64, device=q.device)] + ([torch.zeros_like(x) for x in (q, k, v)] if c["backward"] else [])
    place = torch.arange(S - T, S, device=q.device).double()
    keys = torch.arange(S, device=q.device).double()
    for b in range(B):
        if c["causal"]:
            front = float(s["prefix"][b]) if s["prefix"] is not None else 0.0
            hidden = (keys[None, :] > place[:, None]) & (keys[None, :] >= front)
        else:
            hidden = torch.zeros(T, S, dtype=torch.bool, device=q.device)
        if s["doc"] is not None:
            mine, theirs = s["doc"][b, S - T:], s["doc"][b]
            hidden = hidden | (mine[:, None] != theirs[None, :]) | (mine < 0)[:, None]
        for h in range(H):
            x = [y.clone().requires_grad_(c["backward"]) for y in (q[b, :, h], k[b, :, h // (H // Hk)], v[b, :, h // (H // Hk)])]
            score = -sum((x[0][:, None, w0:w0 + 8] - x[1][None, :, w0:w0 + 8]).abs().sum(2) for w0 in range(0, c["W"], 8)) / c["W"] ** 0.5
            if c["cap"]:
                score = c["cap"] * torch.tanh(score / c["cap"])
            if s["slopes"]:
                score = score - s["slopes"][h] * (place[:, None] - keys[None, :]).abs()
            score = torch.cat([score.masked_fill(hidden, -float("inf")), torch.zeros(T, 1, dtype=torch.float64, device=q.device)], 1)
            o = torch.softmax(score, 1)[:, :S] @ x[2]
            out[0][b, :, h] = o.detach()
            if c["backward"]:
                gq, gk, gv = torch.autograd.grad(o, x, s["do"][b, :, h].double())
                out[1][b, :, h] = gq
                out[2][b, :, h // (H // Hk)] += gk
                out[3][b, :, h // (H // Hk)] += gv
    return out


def _exact_attend(s):
    c, pool = s["case"], s["pool"]
    B, n, H, Hk, P = (c[k] for k in ("B", "n", "H", "Hk", "page"))
    q = s["q"].double()
    out = torch.zeros(B, n, H, c["Wv"], dtype=torch.float64, device=q.device)
    for b, length in enumerate(pool["lens"][:B].tolist()):
        pages = pool["table"][b, :(length + P - 1) // P].long()
        k, v = ((pool[a + "_pages"][pages].double() * pool[a + "_scale"][pages].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :length] for a in "kv")
        for j in range(n):
            m = length - n + j + 1  # tokens that this query sees
            x = q[b, j].view(Hk, H // Hk, 1, -1) - k[:, None, :m]
            x = -x.abs().sum(-1) / c["W"] ** 0.5
            if c["cap"]:
                x = torch.tanh(x / c["cap"]) * c["cap"]
            if s["slopes"]:
                far = torch.arange(m - 1, -1, -1, device=q.device).double()
                x = x - torch.tensor(s["slopes"], dtype=torch.float64, device=q.device).view(Hk, -1, 1) * far
            x = torch.softmax(torch.cat([x, torch.zeros_like(x[..., :1])], -1), -1)[..., :m]
            out[b, j] = (x @ v[:, :m]).reshape(H, -1)
    return [out]


def _exact_scales(s, a):
    """The pool's scales after append(): the largest magnitude of a page's new values over 127, or the one it had."""
    pool, P = s["pool"], s["case"]["page"]
    scale = pool[a + "_scale"].double().clone()
    top = int(pool["n_free"])
    for b in range(s["case"]["B"]):
        start, count = int(pool["lens"][b]), int(s["counts"][b])
        for p in range(start // P, (start + count + P - 1) // P):
            lo, hi = max(start, p * P), min(start + count, (p + 1) * P)
            largest = s[a][b, lo - start:hi - start].double().abs().amax((0, 2)) / 127
            if p * P < start:
                page = int(pool["table"][b, p])
                scale[page] = torch.maximum(scale[page], largest)
            else:
                top -= 1
                scale[int(pool["free"][top])] = largest
    return scale


def _exact_fork_scales(s, a):
    """The pool's scales after the forks' append(): a child's first page is a copy of its parent's with new tokens behind, or a new one."""
    c, pool = s["case"], s["pool"]
    P, n = c["page"], c["n"]
    scale = pool[a + "_scale"].double().clone()
    top = int(pool["n_free"])
    lens = pool["lens"].tolist()
    for r, parent in enumerate(s["parents"].tolist()):
        start = lens[parent]
        for p in range(start // P, (start + n + P - 1) // P):
            lo, hi = max(start, p * P), min(start + n, (p + 1) * P)
            largest = s[a][r, lo - start:hi - start].double().abs().amax((0, 2)) / 127
            if p * P < start:
                largest = torch.maximum(largest, pool[a + "_scale"][int(pool["table"][parent, p])].double())
            top -= 1
            scale[int(pool["free"][top])] = largest
    return scale
