"""CPU-only: what the paged cache and its attention refuse before anything is launched, and their plain model's own checks."""
import ctypes

import pytest
import torch

import _l1attn_lm_hip as drv
import lm_forms as lf


@pytest.fixture()
def no_gpu(monkeypatch):
    monkeypatch.setattr(drv, "check_input", lambda x, name: None)


def _cache(W=16, **kw):
    import l1attn_paged_cuda as m
    return m.L1PagedCache.empty(4, 16, 2, W, 3, 5, device="cpu", **kw)


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        _cache()


def test_state_is_checked(no_gpu):
    import l1attn_paged_cuda as m
    c = _cache()
    good = dict(k_pages=c.k_pages, v_pages=c.v_pages, k_scale=c.k_scale, v_scale=c.v_scale, table=c.table, lens=c.lens, refs=c.refs, free=c.free_pages,
                n_free=c.n_free)
    m.L1PagedCache(**good)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for what in (dict(k_pages=c.k_pages.float()), dict(v_pages=c.v_pages[:3]), dict(k_scale=torch.zeros(4, 3)), dict(v_scale=torch.zeros(4, 2).double()),
                 dict(table=i(3)), dict(lens=i(4)), dict(refs=i(3)), dict(free=i(5)), dict(n_free=i(2)), dict(width=17), dict(width=0), dict(v_width=129),
                 dict(k_pages=torch.zeros(4, 2, 24, 16, dtype=torch.int8), v_pages=torch.zeros(4, 2, 24, 16, dtype=torch.int8)),
                 dict(table=torch.zeros(3, 5, dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            m.L1PagedCache(**{**good, **what})
    odd = torch.zeros(4 * 2 * 16 * 16 + 1, dtype=torch.int8)[1:].view(4, 2, 16, 16)
    with pytest.raises(RuntimeError, match="16 bytes"):
        m.L1PagedCache(**{**good, "k_pages": odd})


def test_state_is_not_exchanged(no_gpu):
    c = _cache()
    with pytest.raises(AttributeError, match="in place"):
        c.lens = torch.zeros_like(c.lens)
    c.lens.copy_(torch.ones_like(c.lens))
    assert c.lens.tolist() == [1, 1, 1]


def test_calls_are_checked(no_gpu):
    import l1attn_paged_cuda as m
    c = _cache()
    z = lambda *s: torch.zeros(*s)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for k, v in ((z(2, 1, 2, 15), z(2, 1, 2, 16)), (z(2, 1, 3, 16), z(2, 1, 3, 16)), (z(2, 1, 2, 16), z(2, 2, 2, 16)), (z(2, 2, 16), z(2, 2, 16)),
                 (z(2, 1, 2, 16), z(2, 1, 2, 16).half()), (z(2, 1, 2, 16).double(), z(2, 1, 2, 16).double()), (z(4, 1, 2, 16), z(4, 1, 2, 16)),
                 (z(1025, 1, 2, 16), z(1025, 1, 2, 16))):
        with pytest.raises(RuntimeError):
            c.append(k, v)
    for kw in (dict(seqs=i(3)), dict(seqs=i(2).long()), dict(counts=i(1)), dict(counts=z(2))):
        with pytest.raises(RuntimeError):
            c.append(z(2, 1, 2, 16), z(2, 1, 2, 16), **kw)
        with pytest.raises(RuntimeError):
            m.l1attn_paged(z(2, 1, 4, 16), c, **kw)
    for a in ((i(2), i(3)), (i(2, 1), i(2, 1)), (i(2).long(), i(2))):
        with pytest.raises(RuntimeError):
            c.fork(*a)
    with pytest.raises(RuntimeError):
        c.free(i(2), keep=i(3))
    for q in (z(2, 1, 3, 16), z(2, 1, 4, 15), z(2, 4, 16), z(4, 1, 4, 16), z(2, 1, 4, 16).double()):
        with pytest.raises(RuntimeError):
            m.l1attn_paged(q, c)
    with pytest.raises(ValueError, match="slopes"):
        m.l1attn_paged(z(2, 1, 4, 16), c, slopes=(1.0,))
    with pytest.raises(ValueError, match="slopes"):
        m.l1attn_paged(z(2, 1, 2, 16), c, slopes=(1.0, -1.0))
    with pytest.raises(ValueError, match="softcap"):
        m.l1attn_paged(z(2, 1, 4, 16), c, softcap=-2.0)
    with pytest.raises(RuntimeError, match="no gradient"):
        m.l1attn_paged(z(2, 1, 4, 16).requires_grad_(), c)


def test_c_entry_codes():
    L = drv.lib()
    p = 4096  # never read: every call here is refused before a launch

    def cache(**kw):
        d = dict(n_pages=4, page=16, Hk=2, W=16, Wv=16, rows=3, row_pages=5)
        d.update({n: p for n in ("k_pages", "v_pages", "k_scale", "v_scale", "table", "lens", "refs", "free_pages", "n_free")})
        d.update(kw)
        return drv.CacheDesc(**d)

    def append(c, dtype=0, k=p, B=1, n=1, served=p, ws=p, nb=1 << 20):
        return L.l1attn_cache_append(ctypes.addressof(c) if c else None, dtype, k, p, None, None, B, n, served, ws, nb, None)
    assert append(None) == -1
    for kw in (dict(page=24), dict(page=0), dict(Hk=0), dict(W=0), dict(rows=-1), dict(k_pages=None), dict(refs=None), dict(n_free=None), dict(lens=None),
               dict(k_pages=p + 8)):
        assert append(cache(**kw)) == -1, kw
    for kw in (dict(W=129), dict(Wv=129), dict(n_pages=1 << 29), dict(row_pages=1 << 25), dict(rows=1 << 25)):
        assert append(cache(**kw)) == -3, kw
    c = cache()
    assert append(c, dtype=3) == -1 and append(c, B=-1) == -1 and append(c, k=None) == -1 and append(c, served=None) == -1
    assert append(c, B=1025) == -3 and append(c, B=0) == 0
    need = L.l1attn_cache_append_workspace_bytes(ctypes.addressof(c), 1, 1)
    assert need == 16 + 2 * 4 and append(c, nb=need - 1) == -2 and append(c, ws=None) == -2
    a = ctypes.addressof(c)
    assert L.l1attn_cache_fork(a, p, p, 1, p, p, 3, None) == -2 and L.l1attn_cache_fork(a, None, p, 1, p, p, 4, None) == -1
    assert L.l1attn_cache_fork(a, p, p, 2000, p, p, 1 << 20, None) == -3 and L.l1attn_cache_fork(a, p, p, 0, p, p, 0, None) == 0
    assert L.l1attn_cache_free(a, p, p, 1, p, 0, None) == -2 and L.l1attn_cache_free(a, p, p, -1, p, 0, None) == -1
    assert L.l1attn_cache_compact(a, p, p, 0, None) == -2 and L.l1attn_cache_compact(a, None, p, 1 << 20, None) == -1

    def attend(q=p, o=p, ws=p, nb=1 << 30, **kw):
        d = drv.AttendDesc(**{**dict(B=1, n=1, H=4, dtype=0, softcap=0.0, slopes=None), **kw})
        return L.l1attn_cache_attend(a, ctypes.addressof(d), q, None, None, o, ws, nb, None)
    assert L.l1attn_cache_attend(a, None, p, None, None, p, p, 1 << 20, None) == -1
    for kw in (dict(H=3), dict(H=0), dict(B=-1), dict(dtype=3), dict(softcap=-1.0), dict(q=None), dict(o=None)):
        assert attend(**kw) == -1, kw
    for kw in (dict(H=512), dict(B=70000), dict(n=1 << 20)):
        assert attend(**kw) == -3, kw
    assert attend(B=0) == 0 and attend(n=0) == 0


def test_appends_past_a_launch_are_refused():
    # a workgroup of 256 threads for each page of each entry, 2^32 - 1 threads at most: refused while the cache is as it was
    L = drv.lib()
    p = 4096  # never read
    c = drv.CacheDesc(n_pages=4, page=16, Hk=2, W=16, Wv=16, rows=64, row_pages=5,
                      **{n: p for n in ("k_pages", "v_pages", "k_scale", "v_scale", "table", "lens", "refs", "free_pages", "n_free")})
    a = ctypes.addressof(c)
    for B, n, rc in ((64, 16 * ((1 << 18) - 1), -3), (1, 1 << 28, -3), (64, 16 * ((1 << 18) - 2), -2)):
        assert L.l1attn_cache_append(a, 1, p, p, None, None, B, n, p, p, 0, None) == rc, (B, n)


def test_the_plain_model_keeps_its_pages_together():
    import random
    r = random.Random(1)
    c = lf.PlainCache(30, 16, 1, 4, 4, 5, 6)
    g = torch.Generator().manual_seed(0)
    for _ in range(200):
        seqs = r.sample(range(5), r.randint(1, 5))
        what = r.randrange(4)
        if what == 0:
            n = r.randint(1, 40)
            c.append(torch.randn(len(seqs), n, 1, 4, generator=g), torch.randn(len(seqs), n, 1, 4, generator=g), seqs)
        elif what == 1:
            c.fork([r.randrange(5) for _ in seqs], seqs)
        elif what == 2:
            c.free(seqs, [r.randint(0, 80) for _ in seqs])
        else:
            c.compact()
        held = [0] * c.N
        for s in range(5):
            for j in range(-(-c.lens[s] // 16)):
                held[int(c.table[s, j])] += 1
        assert held == c.refs and sorted(c.stack + [p for p in range(c.N) if held[p]]) == list(range(c.N))
    k, v = torch.randn(1, 50, 1, 4, generator=g), torch.randn(1, 50, 1, 4, generator=g)
    c.free(list(range(5)))
    c.append(k, v, [0])
    for x, y in zip(c.tokens(0), (k, v)):
        assert (x - y[0].double()).abs().max() <= y.abs().max() / 127 / 2 * (1 + 1e-6)


def test_binding_matches_the_header():
    import os
    import test_abi_signatures_cpu as sig
    declared = {n: s for n, s in sig._prototypes(open(os.path.join(sig.ROOT, "include", "l1attn_hip.h")).read(), ";").items()
                if n.startswith(("l1attn_masked_", "l1attn_cache_"))}
    assert len(declared) == 13 and sig._check_binding(drv.lib(), declared, set(declared)) == 13
    # the structs, member by member
    text = sig._strip_comments(open(os.path.join(sig.ROOT, "include", "l1attn_hip.h")).read())
    import re
    for name, cls in (("l1attn_masked_desc", drv.MaskedDesc), ("l1attn_cache", drv.CacheDesc), ("l1attn_attend_desc", drv.AttendDesc)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        members = []
        for line in body.split(";"):
            m = re.match(r"\s*(?:const\s+)?(\w+)\s+(.*)", line.strip(), flags=re.S)
            if m:
                members += [(v.strip().split("*")[-1].strip().split(" ")[-1], ctypes.c_void_p if "*" in v or "*" in m.group(1) else
                             {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "float": ctypes.c_float}[m.group(1)]) for v in m.group(2).split(",")]
        assert members == list(cls._fields_), name
