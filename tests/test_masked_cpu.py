"""CPU-only: what masked attention refuses, at the Python operator and at the C entry, before anything is launched."""
import ctypes

import pytest
import torch

import _l1attn_lm_hip as drv


@pytest.fixture()
def no_gpu(monkeypatch):
    monkeypatch.setattr(drv, "check_input", lambda x, name: None)


def _q(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_host_tensors_and_strides_are_refused():
    import l1attn_masked_cuda as m
    q = _q(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        m.L1AttnMasked()(q, q, q)


@pytest.mark.parametrize("what,match", [
    (dict(k=_q(1, 4, 2, 9)), "q must be"), (dict(v=_q(1, 5, 2, 8)), "q must be"), (dict(k=_q(2, 4, 2, 8), v=_q(2, 4, 2, 8)), "q must be"),
    (dict(k=_q(1, 3, 2, 8), v=_q(1, 3, 2, 8)), "last of the keys"), (dict(k=_q(1, 4, 3, 8), v=_q(1, 4, 3, 8)), "multiple"),
    (dict(k=_q(1, 4, 2, 8).half()), "dtype"), (dict(q=_q(1, 4, 2, 8).double(), k=_q(1, 4, 2, 8).double(), v=_q(1, 4, 2, 8).double()), "float32, float16"),
    (dict(v=_q(1, 4, 2, 129)), "1 to 128"), (dict(v=_q(1, 4, 2, 0)), "1 to 128"),
    (dict(doc=torch.zeros(1, 3, dtype=torch.int32)), "doc"), (dict(doc=torch.zeros(1, 4, dtype=torch.int64)), "doc"),
    (dict(prefix=torch.zeros(2, dtype=torch.int32)), "prefix"),
    (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(slopes=(1.0,)), "slopes")])
def test_refusals(no_gpu, what, match):
    a = dict(q=_q(1, 4, 2, 8), k=_q(1, 4, 2, 8), v=_q(1, 4, 2, 8))
    a.update(what)
    with pytest.raises((RuntimeError, ValueError), match=match):
        drv.masked_forward(**a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_what_a_forward_kept_is_checked(no_gpu, dtype):
    # logarithms alone in float32; for 16 bits, on the next 16 bytes, as many numbers of the type as o has
    q, k, v = _q(1, 3, 2, 8, dtype=dtype), _q(1, 4, 2, 8, dtype=dtype), _q(1, 4, 2, 5, dtype=dtype)
    d = drv._masked_desc(q, k, v, None, None, True, 0.0, None)
    floats, rest = drv._kept(d)
    assert (floats, rest) == ((6, None) if dtype == torch.float32 else (8 + 15, 8))
    o = _q(1, 3, 2, 5, dtype=dtype)
    for bad in (_q(1, 3, 2) if dtype != torch.float32 else _q(7), _q(floats + 1), _q(floats, dtype=torch.float64)):
        with pytest.raises(RuntimeError, match="kept must be"):
            drv.masked_backward(o, q, k, v, o, bad)
    with pytest.raises(RuntimeError, match="d_o must be"):
        drv.masked_backward(o[..., :4], q, k, v, o, _q(floats))


def test_slopes_are_constants_of_the_module():
    import l1attn_masked_cuda as m
    for bad in ((-1.0, 0.0), (float("nan"),), (float("inf"),)):
        with pytest.raises(ValueError, match="slopes"):
            m.L1AttnMasked(slopes=bad)


def test_slopes_are_taken_by_their_values():
    # lists, tuples, tensors, and tensors as elements; an element that was changed in place is a new number
    for slopes in ([0.5, 0.25], (0.5, 0.25), torch.tensor([0.5, 0.25]), torch.tensor([0.5, 0.25]).numpy()):
        assert list(drv._check_rule(2, 0.0, slopes)) == [0.5, 0.25]
    t = (torch.tensor(0.5), torch.tensor(0.25))
    assert list(drv._check_rule(2, 0.0, t)) == [0.5, 0.25]
    t[0].fill_(3.0)
    assert list(drv._check_rule(2, 0.0, t)) == [3.0, 0.25]
    assert drv._check_rule(2, 0.0, None) is None
    with pytest.raises(ValueError, match="slopes"):
        drv._check_rule(2, 0.0, (torch.tensor(-1.0), torch.tensor(0.0)))


def test_c_entry_codes():
    L = drv.lib()
    one = ctypes.c_void_p(16)

    def fwd(q=one, o=one, **kw):
        d = dict(B=1, T=4, S=4, H=2, Hk=2, W=8, Wv=8, dtype=0, causal=1, softcap=0.0)
        d.update(kw)
        slopes = d.pop("slope_values", None)
        desc = drv.MaskedDesc(**d)
        if slopes:
            keep = (ctypes.c_float * len(slopes))(*slopes)
            desc.slopes = ctypes.addressof(keep)
        return L.l1attn_masked_fwd(ctypes.addressof(desc), q, one, one, o, None, None, 0, None)
    assert L.l1attn_masked_fwd(None, one, one, one, one, None, None, 0, None) == -1
    assert fwd(q=None) == -1 and fwd(o=None) == -1
    for kw in (dict(T=5), dict(T=-1), dict(B=-1), dict(H=3), dict(Hk=0), dict(W=0), dict(dtype=3), dict(causal=2), dict(softcap=-1.0),
               dict(softcap=float("nan")), dict(slope_values=(0.5, -1.0)), dict(slope_values=(0.5, float("nan")))):
        assert fwd(**kw) == -1, kw
    for kw in (dict(W=129), dict(Wv=129), dict(H=512), dict(S=1 << 23)):
        assert fwd(**kw) == -3, kw
    assert fwd(B=0) == 0 and fwd(T=0) == 0  # nothing to do
    d = drv.MaskedDesc(1, 100, 500, 2, 2, 8, 8, 0, 1, 0.0, None, None, None)
    n = L.l1attn_masked_fwd_workspace_bytes(ctypes.addressof(d))
    assert n > 0 and n % (100 * 2 * 9 * 4) == 0  # one [B,T,H,Wv+1] for each split
    assert L.l1attn_masked_fwd(ctypes.addressof(d), one, one, one, one, None, None, n, None) == -2
    assert L.l1attn_masked_fwd(ctypes.addressof(d), one, one, one, one, None, one, n - 1, None) == -2
    d = drv.MaskedDesc(1, 4, 4, 2, 2, 8, 8, 0, 1, 0.0, None, None, None)
    n = L.l1attn_masked_bwd_workspace_bytes(ctypes.addressof(d))
    assert n == 256
    assert L.l1attn_masked_bwd(ctypes.addressof(d), *[one] * 9, None, n, None) == -2
    assert L.l1attn_masked_bwd(ctypes.addressof(d), *[one] * 10, n - 1, None) == -2
    assert L.l1attn_masked_bwd(ctypes.addressof(d), one, None, *[one] * 8, n, None) == -1


def test_batches_past_a_launch_are_refused():
    # a launch has 2^32 - 1 threads at most along batch and heads
    L = drv.lib()
    one = ctypes.c_void_p(16)
    for kw in (dict(B=1 << 20, H=16, Hk=16, dtype=1), dict(B=1 << 19, H=16, Hk=1), dict(B=1 << 20, H=16, Hk=16, W=65)):
        d = drv.MaskedDesc(**{**dict(B=1, T=1, S=1, H=2, Hk=2, W=8, Wv=8, dtype=0, causal=1), **kw})
        a = ctypes.addressof(d)
        assert L.l1attn_masked_fwd(a, one, one, one, one, None, None, 0, None) == -3, kw
        assert L.l1attn_masked_bwd(a, *[one] * 10, 1 << 40, None) == -3, kw
        d.B -= 1  # the largest batch: looked at as far as the workspace
        assert L.l1attn_masked_bwd(a, *[one] * 10, 0, None) == -2, kw


def test_the_plain_statement_is_the_framework_s_own():
    # without masks it is what the fused operator's closed form says, and its gradients are autograd's
    import closed_forms as cf
    import lm_forms as lf
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(2, 9, 3, 5, generator=g, dtype=torch.float64) for _ in range(4))
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    o = cf.dense_then_value(q, k, v)
    want = [o, *torch.autograd.grad(o, (q, k, v), do)]
    got, _ = lf.masked(q, k, v, do, causal=False)
    for a, b in zip(got, want):
        assert torch.allclose(a, b.detach(), atol=1e-12)
