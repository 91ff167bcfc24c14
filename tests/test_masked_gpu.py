"""Masked L1 attention on the GPU: forward and gradients against the formulas in 64 bits."""
import pytest
import torch

import lm_forms as lf

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _op(**kw):
    import l1attn_masked_cuda
    return l1attn_masked_cuda.L1AttnMasked(**kw)


def _inputs(B, T, S, H, Hk, W, Wv, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, n, h, w, generator=g) for n, h, w in ((T, H, W), (S, Hk, W), (S, Hk, Wv), (T, H, Wv)))
    return [(x * s).to(dtype).cuda() for x, s in ((q, scale), (k, scale), (v, 1.0), (do, 1.0))]


def _run(q, k, v, do, doc=None, prefix=None, causal=True, cap=0.0, slopes=None):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    o = _op(causal=causal, softcap=cap, slopes=slopes)(q, k, v, doc=doc, prefix=prefix)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]


def _check(q, k, v, do, **kw):
    print("case", tuple(q.shape), tuple(k.shape), v.shape[-1], q.dtype, {n: x for n, x in kw.items() if not torch.is_tensor(x)}, flush=True)
    ref, terms = lf.masked(q, k, v, do, **kw)
    got = _run(q, k, v, do, **kw)
    lf.check(got, ref, terms, q.dtype, q.shape[-1])
    return got


def _docs(B, S, n, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, S + 1, (B, n), generator=g).sort(1).values
    doc = (torch.arange(S)[None, :, None] >= cuts[:, None]).sum(2).to(torch.int32)
    if pad:
        doc[:, -pad:] = -1
    return doc.cuda()


SLOPES = lambda H: tuple(2.0 ** (-8 * (h + 1) / H) for h in range(H))  # noqa: E731


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,T,S,H,Hk,W,Wv", [(1, 1, 1, 1, 1, 1, 1), (2, 1, 70, 4, 2, 32, 32), (1, 33, 33, 2, 1, 33, 65), (2, 64, 129, 4, 4, 64, 64),
                                            (1, 65, 200, 3, 1, 65, 33), (1, 130, 130, 2, 2, 96, 128), (1, 100, 100, 2, 1, 128, 7),
                                            (1, 257, 300, 8, 2, 64, 64), (1, 40, 90, 2, 2, 7, 128), (3, 31, 63, 2, 2, 16, 16)])
def test_sizes(B, T, S, H, Hk, W, Wv, dtype):
    _check(*_inputs(B, T, S, H, Hk, W, Wv, dtype, T + S + W))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rule", ["open", "docs", "docs_open", "prefix", "prefix_docs", "cap", "slopes", "all"])
def test_masks(rule, dtype):
    B, T, S, H, Hk, W = 2, 150, 201, 4, 2, 64
    q, k, v, do = _inputs(B, T, S, H, Hk, W, 48, dtype, 5)
    kw = {}
    if "docs" in rule or rule == "all":
        kw["doc"] = _docs(B, S, 5, 3, pad=9)
    if "open" in rule:
        kw["causal"] = False
    if "prefix" in rule or rule == "all":
        kw["prefix"] = torch.tensor([0, 130], dtype=torch.int32).cuda()
    if rule in ("cap", "all"):
        kw["cap"] = 5.0
    if rule in ("slopes", "all"):
        kw["slopes"] = SLOPES(H)
    _check(q, k, v, do, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_documents_in_no_order_and_rows_that_see_nothing(dtype):
    B, T, H, W = 2, 140, 2, 32
    q, k, v, do = _inputs(B, T, T, H, 1, W, W, dtype, 8)
    g = torch.Generator().manual_seed(1)
    doc = torch.randint(-1, 3, (B, T), generator=g).to(torch.int32)
    doc[1] = -1  # a whole sequence of padding
    got = _check(q, k, v, do, doc=doc.cuda(), causal=False)
    for x in got:
        assert (x[1] == 0).all()
    assert (got[0].cpu()[0][doc[0] < 0] == 0).all() and (got[1].cpu()[0][doc[0] < 0] == 0).all()
    assert (got[2].cpu()[0][doc[0] < 0] == 0).all() and (got[3].cpu()[0][doc[0] < 0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_hidden_may_hold_anything(bad, dtype):
    B, T, H, W = 1, 130, 2, 64
    q, k, v, do = _inputs(B, T, T, H, 1, W, W, dtype, 9)
    doc = torch.zeros(B, T, dtype=torch.int32)
    doc[:, 100:] = -1  # padding behind, in the middle of a tile
    doc[:, 40:50] = -1  # and in between
    hidden = doc[0] < 0
    for x in (q, k, v, do):
        x[0, hidden.cuda()] = bad
    got = _check(q, k, v, do, doc=doc.cuda())
    for x in got[1:]:
        assert (x.cpu()[0][hidden] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_what_is_visible_may_be_infinite(causal, dtype):
    # a weight is not zero at these distances: infinity, as of the formula, in the rows that see it, and in no other place
    q, k, v, do = _inputs(1, 100, 100, 2, 2, 32, 48, dtype, 21)
    ref, terms = lf.masked(q, k, v, causal=causal)
    v[0, 70, 1, 5], v[0, 3, 0, 7] = float("inf"), -float("inf")
    o = _op(causal=causal)(q, k, v).double().cpu()
    want = ref[0]
    want[0, 70 if causal else 0:, 1, 5] = float("inf")
    want[0, 3 if causal else 0:, 0, 7] = -float("inf")
    inf = torch.isinf(want)
    assert torch.equal(o[inf], want[inf])
    lf.check([o.where(~inf, torch.zeros(())).to(dtype)], [want.where(~inf, torch.zeros((), dtype=torch.float64))], terms, dtype, 32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_future_may_hold_anything(dtype):
    # values behind a query's own place: not finite, and yet not seen by the rows before them
    q, k, v, do = _inputs(1, 80, 80, 2, 2, 32, 32, dtype, 10)
    clean = _run(q, k, v, do)[0]
    k2, v2 = k.clone(), v.clone()
    k2[0, 70:], v2[0, 70:] = float("nan"), float("inf")
    with torch.no_grad():
        o = _op()(q, k2, v2)
    assert torch.equal(o[0, :70], clean[0, :70])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1e-3, 30.0])
def test_small_and_large_inputs(scale, dtype):
    _check(*_inputs(1, 120, 120, 2, 2, 64, 64, dtype, 11, scale))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [1e3, 1e5, 1e6, 1e8, 1e12, 1e30, 3e38])
def test_large_caps(cap, dtype):
    # the capped score goes to the score itself: an absolute error of the tanh would be multiplied by the cap
    _check(*_inputs(1, 100, 120, 2, 1, 64, 48, dtype, 51, 0.3), cap=cap)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1e-38, 1e-30, 1e-3])
def test_tiny_caps(cap, dtype):
    # keys that equal queries: a distance of zero over a cap whose reciprocal is beyond float32
    q, k, v, do = _inputs(1, 70, 70, 2, 2, 32, 32, dtype, 52)
    k[:, ::3] = q[:, ::3]
    _check(q, k, v, do, cap=cap)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [0.3, 1.0, 2.0])
def test_gradients_of_saturated_caps(cap, dtype):
    # the tanh's derivative is 1e-26 to 1e-2 here, and the gradients have its digits.  The formula's own 1 - (c/cap)^2 is off by
    # 2^-52 in 64 bits; that much of a score's gradient, 1/8 p (|do||v| + 2 |do||o|) with p <= 1, |o| <= max |v| and 32 columns,
    # comes in for each of up to 90 pairs
    q, k, v, do = _inputs(1, 70, 90, 2, 2, 64, 32, dtype, 53)
    ref, terms = lf.masked(q, k, v, do, cap=cap)
    of_the_formula = 2.0 ** -52 * 90 / 8 * 3 * 32 * float(v.abs().max()) * float(do.abs().max())
    for t in terms[1:3]:
        t += of_the_formula / (2.0 ** -24 * (3 * 64 + 64))  # check() multiplies the terms by this
    lf.check(_run(q, k, v, do, cap=cap), ref, terms, dtype, 64)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("slope", [2e38, 2.5e38, 3e38])
def test_largest_slopes(slope, dtype):
    _check(*_inputs(1, 70, 90, 2, 1, 32, 32, dtype, 54), slopes=(slope, 0.25))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shift,W,Wv", [(0.0, 64, 64), (300.0, 64, 64), (0.0, 100, 128)])
def test_a_few_far_values(shift, W, Wv, dtype):
    # one owner row and one streamed row far off the others, and all of them far from zero (exact in 16 bits: quarters)
    q, k, v, do = _inputs(1, 90, 90, 2, 1, W, Wv, dtype, 31)
    q, k = (((x.float() * 2).round() / 4 + shift).to(dtype) for x in (q, k))
    q[0, 40], k[0, 7, :, 3] = 500.0, -500.0
    _check(q, k, v, do)


def _few_values(dtype, rng, W, seed, T=128, H=4):
    # rows of one value, keys at distances that leave a weight; a far pair of columns in every 32 rows makes the range
    g = torch.Generator().manual_seed(seed)
    a = (torch.rand(1, T, H, 1, generator=g) - 0.5) * 0.9 * rng
    q = a.expand(1, T, H, W).clone()
    k = (a + (torch.rand(1, T, H, 1, generator=g) - 0.5) * 8 / W ** 0.5).expand(1, T, H, W).clone()
    for x in (q, k):
        x[:, ::32, :, 0], x[:, 1::32, :, 0] = rng / 2, -rng / 2
    v, do = torch.randn(1, T, H, 32, generator=g), torch.randn(1, T, H, 32, generator=g)
    return [x.to(dtype).cuda() for x in (q, k, v, do)]


@pytest.mark.parametrize("dtype,rng", [(F16, 23.5), (F16, 11.8), (F16, 8.0), (BF16, 158.0), (BF16, 94.0), (BF16, 30.0)])
@pytest.mark.parametrize("W", [16, 64, 96, 128])
def test_rows_of_few_values(W, dtype, rng):
    # a document of its own for each token: one weight alone is in a result, and all columns' roundings in its logit
    q, k, v, do = _few_values(dtype, rng, W, W)
    _check(q, k, v, do, doc=torch.arange(128, dtype=torch.int32)[None].cuda())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("logit", [-14.0, -19.0, -23.0, -25.0, -28.0])
def test_weights_that_are_all_small(logit, dtype):
    # all of a row's weights alike and down to 2^-40, under large values and gradients: results well above the type's smallest numbers
    W, T = 64, 256
    g = torch.Generator().manual_seed(58)
    q = torch.zeros(1, T, 2, W)
    k = torch.full((1, T, 2, W), -logit / W ** 0.5) * (torch.randint(0, 2, (1, T, 2, W), generator=g) * 2 - 1)
    v, do = (2e4 + 3e4 * torch.rand(1, T, 2, 48, generator=g) for _ in range(2))
    do *= 2.0 ** -10
    _check(*(x.to(dtype).cuda() for x in (q, k, v, do)), causal=False)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,T,H,Wv", [(1, 512, 2, 64), (1, 512, 2, 37), (8, 150, 32, 64), (8, 150, 32, 33)])
def test_values_with_a_common_part(B, T, H, Wv, dtype):
    # do . v and do . o nearly cancel.  With u the half step: the gradients' own rounding is u of them at most, so u rms; of the terms
    # (which hold 2 |do||o|) u^2 is what two numbers of the type leave of o, and 32 * 2^-24 covers, rms, float32 sums of up to 512
    # terms (their roundings add as a square root), of 64 differences, and exp.  Far values in each 32 rows keep 16-bit codes out.
    q, k, v, do = _inputs(B, T, T, H, H, 64, Wv, dtype, 55, 0.1)
    v += 16
    q[:, ::32, :, 0], k[:, 1::32, :, 0] = 100.0, 100.0
    got = _run(q, k, v, do)
    u = torch.finfo(dtype).eps / 2
    rms = lambda x: float(x.double().square().mean().sqrt())  # noqa: E731
    for b, h in {(0, 0), (B - 1, H - 1)}:
        ref, terms = lf.masked(*(x[b:b + 1, :, h:h + 1] for x in (q, k, v, do)))
        for n, x, r, t in zip(("dq", "dk"), got[1:3], ref[1:3], terms[1:3]):
            off, room = rms(x[b:b + 1, :, h:h + 1].cpu() - r), u * rms(r) + (u * u + 32 * 2.0 ** -24) * rms(t)
            assert off <= room, "%s: off by %.3g of its size rms where %.3g is allowed" % (n, off / rms(r), room / rms(r))


def test_a_prefix_changes_nothing_without_causal():
    q, k, v, do = _inputs(2, 70, 70, 2, 1, 33, 40, BF16, 32)
    prefix = torch.tensor([30, 0], dtype=torch.int32).cuda()
    for a, b in zip(_run(q, k, v, do, causal=False, prefix=prefix), _run(q, k, v, do, causal=False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_tensor_for_all_and_broadcast_keys(dtype):
    x, _, _, do = _inputs(2, 65, 65, 2, 2, 48, 48, dtype, 33)
    parts = _run(x, x, x, do)
    y = x.detach().requires_grad_()
    got, = torch.autograd.grad(_op()(y, y, y), y, do)
    total = sum(p.double() for p in parts[1:])
    # autograd adds the three in the tensor's type: two roundings, of sums no larger than the parts' magnitudes
    room = 2 * torch.finfo(dtype).eps * sum(p.double().abs() for p in parts[1:]) + 1e-30
    assert ((got.double() - total).abs() <= room).all()
    one = x[:1].detach().requires_grad_()
    g, = torch.autograd.grad(_op()(x, one.expand(2, -1, -1, -1), x), one, do)
    dk = _run(x, x[:1].repeat(2, 1, 1, 1), x, do)[2].double()
    assert ((g.double() - dk.sum(0, keepdim=True)).abs() <= torch.finfo(dtype).eps * dk.abs().sum(0, keepdim=True) + 1e-30).all()


def test_a_captured_training_step_and_two_calls_at_once():
    q, k, v, do = _inputs(2, 130, 130, 4, 2, 64, 64, BF16, 34)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    op = _op(softcap=8.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):  # as a captured step needs it: the first pass on a stream of its own, nothing of it kept
        torch.autograd.grad(op(*leaves), leaves, do)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(op(*leaves), leaves, do)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for seed in range(3):
        fresh = _inputs(2, 130, 130, 4, 2, 64, 64, BF16, 40 + seed)
        with torch.no_grad():
            for a, b in zip(leaves, fresh):
                a.copy_(b)
        want = _run(*fresh[:3], do, cap=8.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want[1:]))
        got = []
        for t in streams:
            t.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(t):
                got.append(_run(*fresh[:3], do, cap=8.0))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x in got for a, b in zip(x, want))


def test_ties_have_no_sign():
    # integers: many pairs are equal in a column, and sign(0) = 0
    g = torch.Generator().manual_seed(2)
    for dtype in (F32, F16, BF16):
        q, k = (torch.randint(-2, 3, (1, 90, 2, 64), generator=g).to(dtype).cuda() for _ in range(2))
        v, do = (torch.randn(1, 90, 2, 64, generator=g).to(dtype).cuda() for _ in range(2))
        _check(q, k, v, do)
        same = torch.ones(1, 50, 1, 32, dtype=dtype, device="cuda")
        out = _run(same, same, torch.randn(1, 50, 1, 32, generator=g).to(dtype).cuda(), torch.ones(1, 50, 1, 32, dtype=dtype, device="cuda"))
        assert out[1].abs().max() <= 1e-5 and out[2].abs().max() <= 1e-5


def test_signs_of_the_smallest_differences():
    # below float32's normal numbers: a difference is a difference
    g = torch.Generator().manual_seed(56)
    q, k = ((torch.randn(1, 60, 2, 32, generator=g) * 1e-40).cuda() for _ in range(2))
    k[:, :, :, ::2] = (torch.randint(-3, 4, (1, 60, 2, 16), generator=g) * 1.5e-45).cuda()
    q[:, :, :, ::4] = 0.0
    v, do = (torch.randn(1, 60, 2, 32, generator=g).cuda() for _ in range(2))
    _check(q, k, v, do)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_unaligned_and_strided_inputs(dtype):
    B, T, H, W = 1, 70, 2, 64
    q, k, v, do = _inputs(B, T, T, H, H, W, W, dtype, 12)
    ref = _run(q, k, v, do)

    def shifted(x):  # contiguous, but starting one element into its storage
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view_as(x)
        return y.copy_(x)
    for a, b in zip(_run(*(shifted(x) for x in (q, k, v, do))), ref):
        assert torch.equal(a, b)
    wide = [torch.cat([x, x], 3)[..., :W] for x in (q, k, v, do)]
    assert not wide[0].is_contiguous()
    for a, b in zip(_run(*wide), ref):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,S,H,Hk,W,Wv", [(130, 130, 32, 32, 16, 24), (300, 300, 32, 32, 24, 16), (290, 333, 32, 16, 40, 72), (270, 270, 32, 32, 72, 40)])
@pytest.mark.parametrize("rule", ["causal", "docs", "prefix"])
def test_wide_workgroups(rule, T, S, H, Hk, W, Wv, dtype):
    # batch and heads that fill the chip: workgroups of four waves, and of eight (float32, widths up to 64), with and without splits,
    # the last one partly filled, over several tiles
    B = 8 if Hk == 32 else 16
    q, k, v, do = _inputs(B, T, S, H, Hk, W, Wv, dtype, T + W)
    kw = {}
    if rule == "docs":
        kw["doc"] = _docs(B, S, 4, 5, pad=11)
    if rule == "prefix":
        kw = dict(prefix=torch.randint(0, S, (B,), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda(), cap=9.0, slopes=SLOPES(H))
    got = _run(q, k, v, do, **kw)
    G = H // Hk
    for b, hk in ((0, 0), (B // 2, Hk // 2), (B - 1, Hk - 1)):
        hs = slice(hk * G, hk * G + G)
        sub = {n: x[b:b + 1] if torch.is_tensor(x) else x[hs] if n == "slopes" else x for n, x in kw.items()}
        ref, terms = lf.masked(q[b:b + 1, :, hs], k[b:b + 1, :, hk:hk + 1], v[b:b + 1, :, hk:hk + 1], do[b:b + 1, :, hs], **sub)
        lf.check([got[0][b:b + 1, :, hs], got[1][b:b + 1, :, hs], got[2][b:b + 1, :, hk:hk + 1], got[3][b:b + 1, :, hk:hk + 1]], ref, terms, dtype, W)


def test_repeats_bit_for_bit_and_large_grids():
    q, k, v, do = _inputs(2, 1100, 1100, 8, 2, 64, 64, BF16, 13)
    doc = _docs(2, 1100, 4, 6)
    a, b = _run(q, k, v, do, doc=doc), _run(q, k, v, do, doc=doc)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    ref, terms = lf.masked(q[:1, :, :4], k[:1, :, :1], v[:1, :, :1], do[:1, :, :4], doc=doc[:1])
    lf.check([a[0][:1, :, :4], a[1][:1, :, :4], a[2][:1, :, :1], a[3][:1, :, :1]], ref, terms, BF16, 64)


@pytest.mark.parametrize("W", [64, 128])
def test_roundings_of_float32_distances(W):
    # One key for each query (a document each) and values of one: o and dv are the weight, whose relative error is the logit's error.
    # A logit x is 1/sqrt(W), as float32, times two sums of W / 8 parts: of a sum, the k-th rounding is 2^-24 / sqrt(3) of k parts at
    # most, rms; with the square root of the sum of squares, and the last product's rounding, 2^-24 |x| sqrt(W / 8 / 18 + 1 / 3), and
    # two more 2^-24 for exp and the rest.  (One sum of W / 4 parts: half as much again.)  The backward of width 64 has one sum.
    g = torch.Generator().manual_seed(60)
    q, k = (3 * torch.randn(1, 256, 8, W, generator=g) for _ in range(2))
    one = torch.ones(1, 256, 8, 4, device="cuda")
    o, _, _, dv = _run(q.cuda(), k.cuda(), one, one, doc=torch.arange(256, dtype=torch.int32)[None].cuda())
    rw = torch.tensor(W ** -0.5, dtype=F32).double()
    x = (q.double() - k.double()).abs().sum(3, keepdim=True) * rw
    want = torch.exp(-x) / (1 + torch.exp(-x))
    room = 2.0 ** -24 * (float(x.square().mean().sqrt()) * (W / 144 + 1 / 3) ** 0.5 + 2)
    for got in (o, dv) if W > 64 else (o,):
        off = float(((got.double().cpu() - want) / want).square().mean().sqrt())
        assert off <= room, (off / 2.0 ** -24, room / 2.0 ** -24)


def test_more_tiles_than_are_classified_at_a_time():
    # 70000 keys: over 1024 tiles of 64
    q, k, v, do = _inputs(1, 3, 70000, 1, 1, 32, 32, F32, 14)
    doc = torch.zeros(1, 70000, dtype=torch.int32)
    doc[:, 100:69000] = 1
    doc[:, 69990:] = 0
    _check(q, k, v, do, doc=doc.cuda())


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(1, 12, 2, 8, generator=g).cuda() for _ in range(4))
    kw = dict(causal=True, cap=4.0, slopes=(0.5, 0.1))
    _, dq, dk, dv = _run(q, k, v, do, **kw)

    def loss(q, k, v):
        return float((lf.masked(q, k, v, **kw)[0][0] * do.double().cpu()).sum())
    eps = 1e-6
    for n, x, d in ((0, q, dq), (1, k, dk), (2, v, dv)):
        for at in ((0, 0, 0, 0), (0, 5, 1, 3), (0, 11, 0, 7), (0, 7, 1, 2)):
            args = [y.double().cpu() for y in (q, k, v)]
            args[n] = args[n].clone()
            args[n][at] += eps
            up = loss(*args)
            args[n][at] -= 2 * eps
            assert abs((up - loss(*args)) / (2 * eps) - float(d[at])) <= 1e-5 + 1e-4 * abs(float(d[at]))


def test_other_streams_and_graph_replays():
    q, k, v, do = _inputs(1, 200, 200, 4, 2, 64, 64, BF16, 15)
    ref = _run(q, k, v, do)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(q, k, v, do)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    import _l1attn_lm_hip as drv
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = drv.masked_forward(q, k, v)
        grads = drv.masked_backward(do, q, k, v, o, lse)
    fresh = _inputs(1, 200, 200, 4, 2, 64, 64, BF16, 16)
    for seed in range(3):
        for x, y in zip((q, k, v, do), fresh):
            x.copy_(torch.roll(y, seed, 1))
        eager = _run(q, k, v, do)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([o, *grads], eager))


def test_empty():
    q = torch.zeros(0, 4, 2, 8, device="cuda", requires_grad=True)
    o = _op()(q, q, q)
    assert o.shape == (0, 4, 2, 8)
    k = torch.randn(1, 5, 2, 8, device="cuda", requires_grad=True)
    q = torch.zeros(1, 0, 2, 8, device="cuda", requires_grad=True)
    o = _op()(q, k, k)
    assert o.shape == (1, 0, 2, 8)
    g = torch.autograd.grad(o, (q, k), torch.zeros_like(o))
    assert g[0].shape == q.shape and (g[1] == 0).all()


def test_a_large_batch_of_small_rows():
    # more than 2^29 rows of queries
    B, T, H = 1048575, 33, 16
    g = torch.Generator(device="cuda").manual_seed(57)
    q, k, v, do = (torch.randn(B, T, H, 1, generator=g, device="cuda", dtype=F16) for _ in range(4))
    got = _run(q, k, v, do)
    for b in (0, B // 2, B - 1):
        ref, terms = lf.masked(*(x[b:b + 1] for x in (q, k, v, do)))
        lf.check([x[b:b + 1] for x in got], ref, terms, F16, 1)


def test_no_queries_for_many_keys():
    # more than 2^32 numbers of dk, on memory that holds others
    k = torch.ones(1, 4194240, 8, 128, dtype=F16, device="cuda")
    ones = torch.ones_like(k)
    del ones
    k.requires_grad_()
    v = torch.ones(1, 4194240, 8, 1, dtype=F16, device="cuda", requires_grad=True)
    q = torch.zeros(1, 0, 8, 128, dtype=F16, device="cuda", requires_grad=True)
    o = _op()(q, k, v)
    for x in torch.autograd.grad(o, (k, v), torch.zeros_like(o)):
        assert not x.any()


def test_it_trains():
    torch.manual_seed(0)
    lin = torch.nn.Linear(32, 3 * 64).cuda()
    x = torch.randn(2, 50, 32, device="cuda")
    q, k, v = lin(x).view(2, 50, 3, 2, 32).unbind(2)
    o = _op(softcap=10.0, slopes=(0.1, 0.2))(q, k, v)
    o.square().mean().backward()
    assert torch.isfinite(lin.weight.grad).all() and lin.weight.grad.abs().max() > 0
