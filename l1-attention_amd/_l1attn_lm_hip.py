"""ctypes binding of the masked attention and of the paged 8-bit cache in libl1attn_hip.so (no counterparts in the reference).

Same contract as the drivers of _l1attn_hip: outputs are allocated here on the caller's current stream and inputs are
borrowed; the cache is the one thing that calls change in place.  Wrong types, shapes and devices raise RuntimeError, wrong
numbers ValueError, before anything is launched.
"""
import ctypes
import functools

import torch

from _l1attn_hip import check, check_input, stream_of
import _l1attn_hip as _hip

_c_p, _c_i64, _c_sz, _c_i = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t, ctypes.c_int
_bound = None


def lib():
    """The HIP library with this module's entry points bound; raises where it is not built."""
    global _bound
    L = _hip.lib()
    if _bound is not L:
        L.l1attn_masked_fwd.restype = _c_i
        L.l1attn_masked_fwd.argtypes = [_c_p] * 7 + [_c_sz, _c_p]
        L.l1attn_masked_fwd_workspace_bytes.restype = _c_sz
        L.l1attn_masked_fwd_workspace_bytes.argtypes = [_c_p]
        L.l1attn_masked_bwd_workspace_bytes.restype = _c_sz
        L.l1attn_masked_bwd_workspace_bytes.argtypes = [_c_p]
        L.l1attn_masked_bwd.restype = _c_i
        L.l1attn_masked_bwd.argtypes = [_c_p] * 11 + [_c_sz, _c_p]
        L.l1attn_cache_append_workspace_bytes.restype = _c_sz
        L.l1attn_cache_append_workspace_bytes.argtypes = [_c_p, _c_i64, _c_i64]
        L.l1attn_cache_append.restype = _c_i
        L.l1attn_cache_append.argtypes = [_c_p, _c_i] + [_c_p] * 4 + [_c_i64, _c_i64, _c_p, _c_p, _c_sz, _c_p]
        L.l1attn_cache_fork.restype = _c_i
        L.l1attn_cache_fork.argtypes = [_c_p] * 3 + [_c_i64, _c_p, _c_p, _c_sz, _c_p]
        L.l1attn_cache_free_workspace_bytes.restype = _c_sz
        L.l1attn_cache_free_workspace_bytes.argtypes = [_c_p]
        L.l1attn_cache_free.restype = _c_i
        L.l1attn_cache_free.argtypes = [_c_p] * 3 + [_c_i64, _c_p, _c_sz, _c_p]
        L.l1attn_cache_compact_workspace_bytes.restype = _c_sz
        L.l1attn_cache_compact_workspace_bytes.argtypes = [_c_p]
        L.l1attn_cache_compact.restype = _c_i
        L.l1attn_cache_compact.argtypes = [_c_p, _c_p, _c_p, _c_sz, _c_p]
        L.l1attn_cache_attend_workspace_bytes.restype = _c_sz
        L.l1attn_cache_attend_workspace_bytes.argtypes = [_c_p, _c_p]
        L.l1attn_cache_attend.restype = _c_i
        L.l1attn_cache_attend.argtypes = [_c_p] * 7 + [_c_sz, _c_p]
        _bound = L
    return L


# ----------------------------------------------------------------------------- masked attention

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class MaskedDesc(ctypes.Structure):
    """l1attn_masked_desc of the C header."""
    _fields_ = [(n, _c_i64) for n in ("B", "T", "S", "H", "Hk", "W", "Wv")] + [
        ("dtype", ctypes.c_int32), ("causal", ctypes.c_int32), ("softcap", ctypes.c_float), ("slopes", _c_p), ("doc", _c_p),
        ("prefix", _c_p), ("o_rest", _c_p)]


def slopes_of(slopes):
    """The distance bias of each head as a tuple of finite numbers >= 0."""
    t = tuple(float(x) for x in slopes)
    if not all(0.0 <= x <= 3e38 for x in t):
        raise ValueError("slopes must be finite numbers >= 0, one for each query head, got %r" % (t[:8],))
    return t


@functools.lru_cache(maxsize=64)
def _slopes_array(slopes):
    return (ctypes.c_float * len(slopes))(*slopes)


def _index_tensor(x, name, shape, q):
    if x is None:
        return None
    if x.dtype != torch.int32 or tuple(x.shape) != shape or x.device != q.device:
        raise RuntimeError("%s must be an int32 tensor of shape %s on the device of q" % (name, list(shape)))
    check_input(x, name)
    return x.data_ptr()


def _check_rule(H, softcap, slopes):
    """The slopes of a call as a C array, or None.  Arrays are kept by the slopes' values: numbers first, since what the caller
    holds may be tensors, which are the same objects when their values are others."""
    if not 0.0 <= softcap <= 3e38:
        raise ValueError("softcap must be a finite number >= 0 (0: none), got %r" % (softcap,))
    if slopes is None:
        return None
    slopes = slopes_of(slopes)
    if len(slopes) != H:
        raise ValueError("slopes must hold one number for each of the %d query heads, got %d" % (H, len(slopes)))
    return _slopes_array(slopes)


def _masked_desc(q, k, v, doc, prefix, causal, softcap, slopes):
    for x, n in ((q, "q"), (k, "k"), (v, "v")):
        check_input(x, n)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] \
            or v.shape[:3] != k.shape[:3]:
        raise RuntimeError("q must be [batch, n_query, n_heads, width], k [batch, n_ctx, n_key_heads, width] and v "
                           "[batch, n_ctx, n_key_heads, value width]")
    if not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device):
        raise RuntimeError("q, k, v must share dtype and device")
    if q.dtype not in DTYPES:
        raise RuntimeError("q: masked attention takes float32, float16 and bfloat16, got %s" % q.dtype)
    B, T, H, W = q.shape
    S, Hk, Wv = k.shape[1], k.shape[2], v.shape[3]
    if T > S:
        raise RuntimeError("the queries are the last of the keys' tokens: n_query %d is more than n_ctx %d" % (T, S))
    if Hk < 1 or H < 1 or H % Hk:
        raise RuntimeError("n_heads must be a multiple of n_key_heads, got %d and %d" % (H, Hk))
    if not (1 <= W <= 128 and 1 <= Wv <= 128):
        raise RuntimeError("widths of masked attention are 1 to 128, got %d and %d" % (W, Wv))
    numbers = _check_rule(H, softcap, slopes)
    d = MaskedDesc(B, T, S, H, Hk, W, Wv, DTYPES[q.dtype], int(bool(causal)), softcap,
                   None if slopes is None else ctypes.addressof(numbers),
                   _index_tensor(doc, "doc", (B, S), q), _index_tensor(prefix, "prefix", (B,), q))
    d.numbers = numbers  # lives as long as the address
    return d


def _kept(d):
    """Floats of what a forward keeps for its backward, and where among them the output's rests begin: [B,T,H] logarithms of the
    denominators, and for 16-bit types, on the next 16 bytes, what the rounding of o left out, as numbers of the type."""
    rows = d.B * d.T * d.H
    rest = -(-rows // 4) * 4
    return (rows, None) if d.dtype == 0 else (rest + -(-rows * d.Wv // 2), rest)


def masked_forward(q, k, v, doc=None, prefix=None, causal=True, softcap=0.0, slopes=None, want_lse=True):
    """Masked L1 attention -> [o, kept]; kept, a row of float32, is what the backward reads (None if not wanted)."""
    d = _masked_desc(q, k, v, doc, prefix, causal, softcap, slopes)
    o = torch.empty((d.B, d.T, d.H, d.Wv), dtype=q.dtype, device=q.device)
    floats, rest = _kept(d)
    kept = torch.empty(floats, dtype=torch.float32, device=q.device) if want_lse else None
    if want_lse and rest is not None:
        d.o_rest = kept.data_ptr() + 4 * rest
    L = lib()
    with torch.cuda.device(q.device):
        n = L.l1attn_masked_fwd_workspace_bytes(ctypes.addressof(d))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        rc = L.l1attn_masked_fwd(ctypes.addressof(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                 None if kept is None else kept.data_ptr(), ws.data_ptr() if n else None, n, stream_of(q))
    check(rc, "l1attn_masked_fwd")
    return [o, kept]


def masked_backward(d_o, q, k, v, o, kept, doc=None, prefix=None, causal=True, softcap=0.0, slopes=None):
    """Gradients of masked_forward -> [dq, dk, dv] from its o and what it kept."""
    d = _masked_desc(q, k, v, doc, prefix, causal, softcap, slopes)
    for x, n in ((d_o, "d_o"), (o, "o"), (kept, "kept")):
        check_input(x, n)
    shape = (d.B, d.T, d.H, d.Wv)
    for x, n in ((d_o, "d_o"), (o, "o")):
        if tuple(x.shape) != shape or x.dtype != q.dtype or x.device != q.device:
            raise RuntimeError("%s must be [batch, n_query, n_heads, value width] with the dtype and device of q" % n)
    floats, rest = _kept(d)
    if tuple(kept.shape) != (floats,) or kept.dtype != torch.float32 or kept.device != q.device:
        raise RuntimeError("kept must be the %d float32 numbers that the forward returned beside o" % floats)
    if rest is not None:
        d.o_rest = kept.data_ptr() + 4 * rest
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    L = lib()
    with torch.cuda.device(q.device):
        n = L.l1attn_masked_bwd_workspace_bytes(ctypes.addressof(d))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        rc = L.l1attn_masked_bwd(ctypes.addressof(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), kept.data_ptr(),
                                 d_o.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n, stream_of(q))
    check(rc, "l1attn_masked_bwd")
    return [dq, dk, dv]


# ------------------------------------------------------------------------------ paged 8-bit cache

class CacheDesc(ctypes.Structure):
    """l1attn_cache of the C header."""
    _fields_ = [(n, _c_i64) for n in ("n_pages", "page", "Hk", "W", "Wv", "rows", "row_pages")] + [
        (n, _c_p) for n in ("k_pages", "v_pages", "k_scale", "v_scale", "table", "lens", "refs", "free_pages", "n_free")]


class AttendDesc(ctypes.Structure):
    """l1attn_attend_desc of the C header."""
    _fields_ = [("B", _c_i64), ("n", _c_i64), ("H", _c_i64), ("dtype", ctypes.c_int32), ("softcap", ctypes.c_float),
                ("slopes", _c_p)]


CACHE_ROWS = 1024  # entries of a list that one call of append, fork or free takes


def _row_list(x, name, B, device):
    """An int32 list of a call as a pointer, or None."""
    if x is None:
        return None
    if x.dtype != torch.int32 or x.dim() != 1 or x.shape[0] != B or x.device != device:
        raise RuntimeError("%s must be an int32 tensor of %d numbers on the cache's device" % (name, B))
    check_input(x, name)
    return x.data_ptr()


def _call_rows(B, rows, listed, name):
    if B > CACHE_ROWS:
        raise RuntimeError("one call serves at most %d sequences, got %d" % (CACHE_ROWS, B))
    if not listed and B > rows:
        raise RuntimeError("%s: %d sequences without a list, but the cache has %d rows" % (name, B, rows))


def cache_append(desc, device, k, v, seqs=None, counts=None):
    """New tokens k [B,n,Hk,W], v [B,n,Hk,Wv] behind the sequences -> served (bool [B]).  desc: the cache's CacheDesc."""
    for x, n in ((k, "k"), (v, "v")):
        check_input(x, n)
        if x.device != device:
            raise RuntimeError("%s must be on the cache's device" % n)
    if k.dim() != 4 or v.dim() != 4 or tuple(k.shape[2:]) != (desc.Hk, desc.W) or tuple(v.shape) != tuple(k.shape[:2]) + (desc.Hk, desc.Wv):
        raise RuntimeError("k must be [batch, n, %d, %d] and v [batch, n, %d, %d]" % (desc.Hk, desc.W, desc.Hk, desc.Wv))
    if k.dtype != v.dtype or k.dtype not in DTYPES:
        raise RuntimeError("k and v must both be float32, float16 or bfloat16, got %s and %s" % (k.dtype, v.dtype))
    B, n = k.shape[:2]
    _call_rows(B, desc.rows, seqs is not None, "append")
    sp, cp = _row_list(seqs, "seqs", B, device), _row_list(counts, "counts", B, device)
    served = torch.empty(B, dtype=torch.bool, device=device)
    L, d = lib(), ctypes.addressof(desc)
    with torch.cuda.device(device):
        nb = L.l1attn_cache_append_workspace_bytes(d, B, n)
        ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=device)
        rc = L.l1attn_cache_append(d, DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), sp, cp, B, n, served.data_ptr(), ws.data_ptr(), nb,
                                   stream_of(k))
    check(rc, "l1attn_cache_append")
    return served


def cache_fork(desc, device, parents, children):
    """Rows children [m] share the pages of rows parents [m] -> served (bool [m])."""
    B = parents.shape[0] if parents.dim() == 1 else -1
    _call_rows(B, desc.rows, True, "fork")
    pp, cp = _row_list(parents, "parents", B, device), _row_list(children, "children", B, device)
    served = torch.empty(B, dtype=torch.bool, device=device)
    with torch.cuda.device(device):
        ws = torch.empty(max(4 * B, 16), dtype=torch.uint8, device=device)
        rc = lib().l1attn_cache_fork(ctypes.addressof(desc), pp, cp, B, served.data_ptr(), ws.data_ptr(), 4 * B, stream_of(parents))
    check(rc, "l1attn_cache_fork")
    return served


def cache_free(desc, device, seqs, keep=None):
    """Sequences seqs [m] keep their first keep [m] tokens, or none."""
    B = seqs.shape[0] if seqs.dim() == 1 else -1
    _call_rows(B, desc.rows, True, "free")
    sp, kp = _row_list(seqs, "seqs", B, device), _row_list(keep, "keep", B, device)
    L, d = lib(), ctypes.addressof(desc)
    with torch.cuda.device(device):
        nb = L.l1attn_cache_free_workspace_bytes(d)
        ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=device)
        rc = L.l1attn_cache_free(d, sp, kp, B, ws.data_ptr(), nb, stream_of(seqs))
    check(rc, "l1attn_cache_free")


def cache_compact(desc, device):
    """The pages in use to the front of the pool -> how many there are (int32 [1])."""
    L, d = lib(), ctypes.addressof(desc)
    live = torch.empty(1, dtype=torch.int32, device=device)
    with torch.cuda.device(device):
        nb = L.l1attn_cache_compact_workspace_bytes(d)
        ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=device)
        rc = L.l1attn_cache_compact(d, live.data_ptr(), ws.data_ptr(), nb, stream_of(live))
    check(rc, "l1attn_cache_compact")
    return live


def cache_attend(desc, device, q, seqs=None, counts=None, softcap=0.0, slopes=None):
    """L1 attention of q [B,n,H,W], the last tokens of the sequences, over the cache -> o [B,n,H,Wv]."""
    check_input(q, "q")
    if q.device != device:
        raise RuntimeError("q must be on the cache's device")
    if q.dim() != 4 or q.shape[3] != desc.W or q.shape[2] < 1 or q.shape[2] % desc.Hk:
        raise RuntimeError("q must be [batch, n, n_heads, %d] with n_heads a multiple of the cache's %d key heads" % (desc.W, desc.Hk))
    if q.dtype not in DTYPES:
        raise RuntimeError("q: paged attention takes float32, float16 and bfloat16, got %s" % q.dtype)
    B, n, H, _ = q.shape
    if seqs is None and B > desc.rows:
        raise RuntimeError("attend: %d sequences without a list, but the cache has %d rows" % (B, desc.rows))
    numbers = _check_rule(H, softcap, slopes)
    sp, cp = _row_list(seqs, "seqs", B, device), _row_list(counts, "counts", B, device)
    a = AttendDesc(B, n, H, DTYPES[q.dtype], softcap, None if slopes is None else ctypes.addressof(numbers))
    o = torch.empty((B, n, H, desc.Wv), dtype=q.dtype, device=device)
    L, d, ap = lib(), ctypes.addressof(desc), ctypes.addressof(a)
    with torch.cuda.device(device):
        nb = L.l1attn_cache_attend_workspace_bytes(d, ap)
        ws = torch.empty(nb, dtype=torch.uint8, device=device) if nb else None
        rc = L.l1attn_cache_attend(d, ap, q.data_ptr(), sp, cp, o.data_ptr(), ws.data_ptr() if nb else None, nb, stream_of(q))
    check(rc, "l1attn_cache_attend")
    return o
