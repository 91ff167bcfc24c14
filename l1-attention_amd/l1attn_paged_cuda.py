"""L1 attention for serving: a paged cache of keys and values in 8 bits, and the attention that reads it, computed by the gfx950
HIP library.  No counterpart in the reference.

    cache = L1PagedCache.empty(n_pages=4096, page=32, n_key_heads=4, width=64, n_rows=64, row_pages=128)
    served = cache.append(k, v, seqs=seqs)          # k [B,n,Hk,W], v [B,n,Hk,Wv]: a prompt, or a step's token
    o = l1attn_paged(q, cache, seqs=seqs)           # q [B,n,H,W]: the last n tokens of each sequence over all of it
    cache.fork(parents, children)                   # children share the parents' pages; a page is copied when it is written to
    cache.free(seqs, keep=lengths)                  # drafted tokens given back; without keep: the whole sequence
    live = cache.compact()                          # pages in use to the front of the pool

A page holds `page` (16, 32 or 64) tokens of every key head as int8 codes; each page and head has a scale, its values' largest
magnitude over 127: value = code * scale.  New tokens that make a page's scale grow make its old codes rint(code * old / new),
which costs those values up to half a step more.  Infinite values are stored as the largest ones of their page, NaN as zero.

All state lies on the device (see L1PagedCache) and every call is asynchronous and capturable: nothing is read back.  Lists
(seqs, counts, keep, parents, children) are int32 tensors on the device.  append() and fork() return, as a bool tensor, which
entries were served: not where a number is out of range or named before in the list, the pool has no page left or the table's
row no room, a child is not empty or its own parent.  The others are not changed.  Calls that change one cache have to be
ordered on one stream (or by events), as for any tensor that is written in place.
"""
import torch
from torch import nn

import _l1attn_lm_hip as _drv


def _round16(n):
    return -(-n // 16) * 16


class L1PagedCache(object):
    """The state, as tensors that the caller may keep, copy and load (in place):

    k_pages [N,Hk,page,W up to a multiple of 16] and v_pages (with Wv) int8; k_scale, v_scale [N,Hk] float32;
    table [rows,row_pages] int32, the pages of each sequence; lens [rows] int32, its tokens; refs [N] int32, rows that hold the
    page; free [N] int32 with n_free [1] int32, a stack of the pages that nobody holds.  width, v_width: where W is not a
    multiple of 16, its value (codes behind it are zero)."""

    def __init__(self, k_pages, v_pages, k_scale, v_scale, table, lens, refs, free, n_free, width=None, v_width=None):
        N, Hk, page, pk = k_pages.shape if k_pages.dim() == 4 else (0, 0, 0, 0)
        pv = v_pages.shape[-1]
        W, Wv = pk if width is None else width, pv if v_width is None else v_width
        if page not in (16, 32, 64) or Hk < 1 or tuple(v_pages.shape[:3]) != (N, Hk, page):
            raise RuntimeError("k_pages and v_pages must be [n_pages, n_key_heads, 16, 32 or 64 tokens, width]")
        if not (1 <= W <= 128 and 1 <= Wv <= 128) or pk != _round16(W) or pv != _round16(Wv):
            raise RuntimeError("widths of the cache are 1 to 128, its rows the next multiple of 16, got %d in %d and %d in %d" % (W, pk, Wv, pv))
        rows, row_pages = table.shape if table.dim() == 2 else (-1, -1)
        for x, n, dtype, shape in ((k_pages, "k_pages", torch.int8, None), (v_pages, "v_pages", torch.int8, None),
                                   (k_scale, "k_scale", torch.float32, (N, Hk)), (v_scale, "v_scale", torch.float32, (N, Hk)),
                                   (table, "table", torch.int32, (rows, row_pages)), (lens, "lens", torch.int32, (rows,)),
                                   (refs, "refs", torch.int32, (N,)), (free, "free", torch.int32, (N,)), (n_free, "n_free", torch.int32, (1,))):
            _drv.check_input(x, n)
            if x.dtype != dtype or (shape is not None and tuple(x.shape) != shape) or x.device != k_pages.device:
                raise RuntimeError("%s must be a %s tensor%s on the device of k_pages" % (n, dtype, "" if shape is None else " of shape %s" % (list(shape),)))
        if N < 1:
            raise RuntimeError("a cache has one page at least")
        if (k_pages.data_ptr() | v_pages.data_ptr()) & 15:
            raise RuntimeError("k_pages and v_pages must start on 16 bytes")
        self.k_pages, self.v_pages, self.k_scale, self.v_scale = k_pages, v_pages, k_scale, v_scale
        self.table, self.lens, self.refs, self.free_pages, self.n_free = table, lens, refs, free, n_free
        self.device = k_pages.device
        self._desc = _drv.CacheDesc(N, page, Hk, W, Wv, rows, row_pages, *(x.data_ptr() for x in (
            k_pages, v_pages, k_scale, v_scale, table, lens, refs, free, n_free)))

    def __setattr__(self, name, value):
        # the kernels go by the tensors' addresses, taken once
        if "_desc" in self.__dict__:
            raise AttributeError("the state of a cache is written in place (%s.copy_(...)), or a new cache is made of other tensors" % name)
        super(L1PagedCache, self).__setattr__(name, value)

    @classmethod
    def empty(cls, n_pages, page, n_key_heads, width, n_rows, row_pages, v_width=None, device=None):
        """A cache of n_pages pages for n_rows sequences of up to row_pages pages each, all of it free."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        v_width = width if v_width is None else v_width
        z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
        return cls(z(n_pages, n_key_heads, page, _round16(width), dtype=torch.int8), z(n_pages, n_key_heads, page, _round16(v_width), dtype=torch.int8),
                   z(n_pages, n_key_heads, dtype=torch.float32), z(n_pages, n_key_heads, dtype=torch.float32),
                   z(n_rows, row_pages) - 1, z(n_rows), z(n_pages), torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=dev),
                   torch.tensor([n_pages], dtype=torch.int32, device=dev), width=width, v_width=v_width)

    def append(self, k, v, seqs=None, counts=None):
        """The first counts[b] (all, without counts) rows of k [B,n,Hk,W] and v [B,n,Hk,Wv] behind sequence seqs[b] (b, without
        seqs) -> served (bool [B]).  A partly filled page that other sequences hold too is copied first."""
        return _drv.cache_append(self._desc, self.device, k.detach().contiguous(), v.detach().contiguous(), seqs, counts)

    def fork(self, parents, children):
        """Sequences children (empty ones) get the pages of parents, as they are before the call -> served (bool)."""
        return _drv.cache_fork(self._desc, self.device, parents, children)

    def free(self, seqs, keep=None):
        """Sequences keep their first keep[b] tokens (none, without keep); their other pages lose a holder."""
        _drv.cache_free(self._desc, self.device, seqs, keep)

    def compact(self):
        """Moves the pages in use to the front of the pool -> how many there are (int32 [1])."""
        return _drv.cache_compact(self._desc, self.device)


def l1attn_paged(q, cache, seqs=None, counts=None, softcap=0.0, slopes=None):
    """o [B,n,H,Wv] of q [B,n,H,W], the last counts[b] (n, without counts) tokens of sequence seqs[b] (b, without seqs): the
    formula of L1AttnMasked, causal, over the whole sequence as the cache holds it.  Rows behind counts[b] and sequences of no
    tokens give zeros.  For serving: there is no gradient.  The same call gives the same bits; a sequence may round differently
    beside others, whose lengths decide how its sums are cut."""
    if torch.is_grad_enabled() and q.requires_grad:
        raise RuntimeError("l1attn_paged has no gradient: call it under torch.no_grad(), or on q.detach()")
    return _drv.cache_attend(cache._desc, cache.device, q.contiguous(), seqs, counts, softcap, slopes)


class L1AttnPaged(nn.Module):
    """l1attn_paged with the rule of a model's layer (see L1AttnMasked)."""

    def __init__(self, softcap=0.0, slopes=None):
        super(L1AttnPaged, self).__init__()
        self.softcap = float(softcap)
        self.slopes = None if slopes is None else _drv.slopes_of(slopes)

    def forward(self, q, cache, seqs=None, counts=None):
        return l1attn_paged(q, cache, seqs, counts, self.softcap, self.slopes)
