"""The paged 8-bit cache and the attention over it on the GPU, against a plain model of both: tables, codes and scales have to be
equal, attention is held to its rounding (lm_forms.check)."""
import pytest
import torch

import lm_forms as lf

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


class Pair:
    """The cache on the GPU beside its plain model; every call goes to both, and their states are compared after it."""

    def __init__(self, N=40, P=16, Hk=2, W=32, Wv=48, rows=6, M=12, dtype=BF16, seed=0):
        import l1attn_paged_cuda as m
        self.m, self.dtype = m, dtype
        self.gpu = m.L1PagedCache.empty(N, P, Hk, W, rows, M, v_width=Wv, device="cuda")
        self.plain = lf.PlainCache(N, P, Hk, W, Wv, rows, M)
        self.g = torch.Generator().manual_seed(seed)

    def data(self, B, n, scale=1.0):
        p = self.plain
        return [(torch.randn(B, n, p.Hk, w, generator=self.g) * scale).to(self.dtype) for w in (p.W, p.Wv)]

    def ints(self, x):
        return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")

    def append(self, B, n, seqs=None, counts=None, scale=1.0, data=None):
        k, v = self.data(B, n, scale) if data is None else data
        got = self.gpu.append(k.cuda(), v.cuda(), seqs=self.ints(seqs), counts=self.ints(counts))
        want = self.plain.append(k, v, seqs, counts)
        assert got.tolist() == want, (got.tolist(), want)
        self.same()
        return want

    def fork(self, parents, children):
        got, want = self.gpu.fork(self.ints(parents), self.ints(children)), self.plain.fork(parents, children)
        assert got.tolist() == want
        self.same()
        return want

    def free(self, seqs, keep=None):
        self.gpu.free(self.ints(seqs), keep=self.ints(keep))
        self.plain.free(seqs, keep)
        self.same()

    def compact(self):
        assert int(self.gpu.compact()) == self.plain.compact()
        self.same()

    def same(self):
        g, p = self.gpu, self.plain
        assert g.lens.tolist() == p.lens
        for s in range(p.rows):
            used = -(-p.lens[s] // p.P)
            assert g.table[s, :used].tolist() == p.table[s, :used].tolist()
        assert g.refs.tolist() == p.refs
        assert g.free_pages[:int(g.n_free)].tolist() == p.stack
        for a, b in ((g.k_scale, p.scale[0]), (g.v_scale, p.scale[1])):
            assert torch.equal(a.cpu(), b)
        for a, b in ((g.k_pages, p.pages[0]), (g.v_pages, p.pages[1])):
            assert torch.equal(a.cpu(), b)

    def attend(self, B, n, H, seqs=None, counts=None, cap=0.0, slopes=None, dtype=None, q=None):
        p, dtype = self.plain, dtype or self.dtype
        q = (torch.randn(B, n, H, p.W, generator=self.g) if q is None else q).to(dtype)
        print("case attend", B, n, H, p.Hk, p.W, p.Wv, p.P, dtype, seqs, counts, cap, flush=True)
        o = self.m.l1attn_paged(q.cuda(), self.gpu, seqs=self.ints(seqs), counts=self.ints(counts), softcap=cap, slopes=slopes)
        ref, terms = p.attend(q, seqs, counts, cap, slopes)
        lf.check([o], [ref], [terms], dtype, p.W, names=("o",))
        return o


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("P", [16, 32, 64])
def test_append_in_all_alignments(P, dtype):
    c = Pair(N=60, P=P, rows=4, M=16, dtype=dtype)
    for n, counts in ((1, None), (5, [5, 0, 3, 9]), (P - 1, None), (P, None), (2 * P + 3, [2 * P + 3, P, -4, 1]), (1, None)):
        c.append(4, n, counts=counts, scale=1 + n % 3)


@pytest.mark.parametrize("W,Wv", [(1, 1), (7, 33), (64, 96), (65, 128), (128, 20)])
def test_append_widths(W, Wv):
    c = Pair(W=W, Wv=Wv, Hk=3, N=30, rows=2, M=8)
    for n in (3, 20, 1, 30):
        c.append(2, n)
        c.attend(2, 1, 3)


def test_scales_grow_and_old_codes_follow():
    c = Pair(rows=1)
    for scale in (0.01, 1.0, 0.1, 50.0, 0.0, 3.0):
        c.append(1, 3, scale=scale)


def test_values_that_are_not_finite_or_zero():
    c = Pair(rows=2, dtype=F32)
    k, v = c.data(2, 5)
    k[0, 1, 0, 3], k[0, 2, 1, 5], v[0, 3, 0, 0], v[0, 4, 1, 1] = float("inf"), float("nan"), -float("inf"), float("nan")
    k[1], v[1] = 0.0, 0.0
    c.append(2, 5, data=(k, v))
    c.attend(2, 1, 2, dtype=F32)
    c.append(2, 4)


def test_rows_that_are_not_served():
    c = Pair(N=10, P=16, rows=6, M=4)
    assert c.append(6, 20, seqs=[3, 3, -1, 6, 0, 5]) == [True, False, False, False, True, True]
    # no room in the row (4 pages hold 64 tokens), and the pool: 6 pages taken, 4 left
    assert c.append(3, 45, seqs=[3, 0, 5], counts=[45, 20, 44]) == [False, True, True]
    assert c.append(4, 16, seqs=[1, 2, 4, 5], counts=[16, 16, 0, 0]) == [True, False, True, True]
    assert c.append(2, 16, seqs=[2, 0], counts=[1, 8]) == [False, True]  # 8 tokens fit the page that is there
    c.free([0, 0, 9, -3])
    c.append(1, 40, seqs=[2])


def test_fork_shares_and_copies_on_write():
    c = Pair(N=40, rows=8, M=10)
    c.append(2, 37, seqs=[0, 1])
    assert c.fork([0, 0, 1, 7, 2, 0, 1, 0], [2, 3, 4, 5, 6, 2, 1, 7]) == [True, True, True, True, True, False, False, True]
    c.append(4, 3, seqs=[2, 0, 3, 4], scale=2.0)
    c.append(1, 3, seqs=[1], scale=0.5)  # the page that 4 left behind has one holder again: written in place
    c.attend(5, 2, 4, seqs=[0, 1, 2, 3, 4])
    c.free([2, 4], keep=[36, 10])
    c.append(2, 30, seqs=[4, 2])
    # all holders of a shared page write to it at once: it is free afterwards
    c.free([0, 1, 2, 3, 4, 7])
    c.append(1, 20, seqs=[0])
    c.fork([0, 0], [1, 2])
    c.append(3, 1, seqs=[2, 0, 1])
    c.attend(3, 1, 2)


def test_free_keeps_a_prefix_and_gives_back_in_order():
    c = Pair(N=40, rows=5, M=10)
    c.append(5, 70, counts=[70, 33, 16, 0, 64])
    c.free([4, 0, 1], keep=[100, 32, 0])
    c.free([2, 3], keep=[16, 5])
    c.append(5, 40)
    c.free([0, 1, 2, 3, 4])


def test_compact_and_going_on():
    c = Pair(N=64, rows=8, M=8)
    c.append(8, 70, counts=[70, 20, 50, 64, 1, 33, 80, 16])
    c.fork([0], [7]) if c.plain.lens[7] == 0 else c.free([7])
    c.fork([0, 2], [7, 6])
    c.free([0, 3, 5])
    c.compact()
    c.attend(8, 1, 2)
    c.append(4, 30, seqs=[0, 3, 7, 5])
    c.compact()
    c.compact()  # nothing moves any more
    c.free(list(range(8)))
    c.compact()
    c.append(8, 30)


def test_pools_of_several_scan_chunks():
    c = Pair(N=9000, P=16, Hk=1, W=16, Wv=16, rows=3, M=4096)
    c.append(2, 40000, counts=[40000, 30000])
    c.free([0], keep=[17])
    c.append(1, 33, seqs=[2])
    c.compact()
    c.append(1, 100, seqs=[2])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Hk,H,n,W,Wv,P", [(1, 1, 1, 32, 32, 16), (2, 4, 1, 64, 64, 32), (2, 2, 3, 33, 65, 64), (1, 8, 1, 96, 128, 16), (2, 16, 5, 64, 64, 32),
                                          (1, 24, 2, 128, 96, 64), (3, 9, 7, 17, 5, 16)])
def test_attention(Hk, H, n, W, Wv, P, dtype):
    c = Pair(N=140, P=P, Hk=Hk, W=W, Wv=Wv, rows=5, M=2200 // P, dtype=dtype, seed=H + W)
    for counts in ([600, 1, 256, 0, 2], [3, 0, 1, 0, 255]):
        c.append(5, 600, counts=counts)
        c.attend(5, n, H)
    slopes = tuple(2.0 ** (-8 * (h + 1) / H) for h in range(H))
    c.attend(4, n, H, seqs=[2, 0, 0, 77], cap=5.0, slopes=slopes)
    c.attend(3, n, H, seqs=[4, 1, 2], counts=[n, 0, max(0, n - 1)], slopes=slopes)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1e-3, 4.0, 30.0])
@pytest.mark.parametrize("H,n,W", [(2, 1, 64), (8, 2, 64), (16, 3, 112)])
def test_small_and_large_inputs(H, n, W, scale, dtype):
    # queries near cached tokens, so that weights are there at every scale; the largest ranges leave the 16-bit codes
    c = Pair(N=60, P=32, Hk=2, W=W, Wv=W, rows=3, M=25, dtype=dtype, seed=n)
    k, v = c.data(3, 700, scale)
    c.append(3, 700, counts=[700, 33, 1], data=(k, v))
    near = k[:, :n].float().repeat_interleave(H // 2, 2)
    c.attend(3, n, H, q=near + 0.1 * scale * torch.randn(near.shape, generator=c.g))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H", [2, 12])
@pytest.mark.parametrize("cap", [1e3, 1e5, 1e6, 1e8, 1e12, 1e30, 3e38])
def test_large_caps(cap, H, dtype):
    c = Pair(N=40, P=16, Hk=2, W=64, Wv=48, rows=2, M=12, dtype=dtype, seed=21)
    c.append(2, 150, counts=[150, 9], scale=0.3)
    c.attend(2, 2, H, cap=cap, q=0.3 * torch.randn(2, 2, H, 64, generator=c.g))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H", [2, 12])
@pytest.mark.parametrize("cap,slope", [(1e-45, 0.0), (1e-39, 0.0), (1e-38, 1.0), (0.3, 0.0), (0.0, 2.5e38), (0.0, 3e38)])
def test_tiny_caps_and_largest_slopes(cap, slope, H, dtype):
    # distances of zero, over a cap whose reciprocal is beyond float32
    c = Pair(N=40, P=16, Hk=2, W=64, Wv=48, rows=2, M=12, dtype=dtype, seed=21)
    k, v = c.data(2, 150, 0.3)
    k[:, :8] = 0.0
    c.append(2, 150, counts=[150, 9], data=(k, v))
    q = 0.3 * torch.randn(2, 2, H, 64, generator=c.g)
    q[1] = 0.0
    c.attend(2, 2, H, cap=cap, q=q, slopes=(slope,) * H)


@pytest.mark.parametrize("dtype,rng", [(F16, 23.5), (F16, 11.8), (F16, 8.0), (BF16, 158.0), (BF16, 94.0), (BF16, 30.0)])
@pytest.mark.parametrize("W", [16, 64, 96, 128])
def test_rows_of_few_values(W, dtype, rng):
    # one token a sequence: its weight alone is in the result
    B, H = 48, 8
    c = Pair(N=64, P=16, Hk=1, W=W, Wv=32, rows=B, M=2, dtype=F32, seed=W)
    top = rng / 2 / 128 * 127 * 0.999  # the grid is over the 128-fold of the scale
    a = (torch.rand(B, 1, 1, 1, generator=c.g) - 0.5) * 2 * top
    k = a.expand(B, 1, 1, W).clone()
    k[:, :, :, 1] = top
    v = torch.randn(B, 1, 1, 32, generator=c.g)
    c.append(B, 1, data=(k, v))
    q = (a + (torch.rand(B, 1, H, 1, generator=c.g) - 0.5) * 8 / W ** 0.5).clamp(-top, top).expand(B, 1, H, W).clone()
    q[:, :, :, 1] = top
    c.attend(B, 1, H, dtype=dtype, q=q)


@pytest.mark.parametrize("B,H,n", [(300, 2, 1), (300, 4, 5), (513, 2, 2)])
def test_many_entries(B, H, n):
    # every row of the table many times, in no order, some that are not there; uneven lengths over several steps
    c = Pair(N=200, P=32, Hk=1, W=64, Wv=64, rows=7, M=40, seed=9)
    c.append(7, 1200, counts=[1200, 0, 1, 513, 256, 800, 40])
    seqs = torch.randint(-1, 8, (B,), generator=c.g).tolist()
    q = torch.randn(7, n, H, 64, generator=c.g).to(BF16)
    each = c.attend(7, n, H, q=q)
    o = c.m.l1attn_paged(torch.stack([q[s % 7] for s in seqs]).cuda(), c.gpu, seqs=c.ints(seqs))
    ref, terms = c.plain.attend(q)
    none = torch.zeros_like(ref[0])
    lf.check([o], [torch.stack([ref[s] if 0 <= s < 7 else none for s in seqs])], [torch.stack([terms[s] if 0 <= s < 7 else none for s in seqs])], BF16, 64, names=("o",))
    assert each.shape == q.shape


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H", [2, 20])
def test_scales_of_hidden_tokens_have_no_influence(H, dtype):
    # a page behind the queries' place, and one that only the padding rows would see, with scales that are not finite
    c = Pair(N=40, P=16, Hk=2, W=64, Wv=64, rows=2, M=8, dtype=dtype)
    c.append(2, 100, counts=[100, 90])
    q = torch.randn(1, 40, H, 64, generator=c.g).to(dtype).cuda()
    want = c.m.l1attn_paged(q, c.gpu)
    if dtype == F16:  # weights times scale that float16 holds only at the right power of two: values up to 2000
        c.gpu.v_scale.mul_(512)
        want = c.m.l1attn_paged(q, c.gpu)
    last = int(c.gpu.table[0, 6])  # tokens 96 to 99: the last four query tokens see them
    c.gpu.k_scale[last], c.gpu.v_scale[last] = float("nan"), float("inf")
    got = c.m.l1attn_paged(q, c.gpu)
    big = 4.5 * (512 if dtype == F16 else 1)
    tol = 2 * (torch.finfo(dtype).eps + 2.0 ** -24 * (3 * 64 + 64)) * big  # both within the bound of lm_forms, of values up to `big`
    assert (got[:, :36].float() - want[:, :36].float()).abs().max() <= tol


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H", [2, 20])
def test_hidden_scales_that_are_large(H, dtype):
    # the last page's values are finite and beyond float16; the tokens before it do not see them
    c = Pair(N=40, P=16, Hk=2, W=64, Wv=64, rows=1, M=8, dtype=F32, seed=3)
    c.append(1, 96)
    k, v = c.data(1, 4)
    c.append(1, 4, data=(k, v * 1e30))
    q = torch.randn(1, 40, H, 64, generator=c.g).to(dtype)
    o = c.m.l1attn_paged(q.cuda(), c.gpu)[:, :36]
    ref, terms = c.plain.attend(q)
    lf.check([o], [ref[:, :36]], [terms[:, :36]], dtype, 64, names=("o",))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H", [2, 20])
def test_visible_infinite_scales(H, dtype):
    # infinity times a code that is not zero, of one sign in each column: infinity, as of the formula
    c = Pair(N=40, P=16, Hk=2, W=64, Wv=64, rows=1, M=8, dtype=dtype, seed=5)
    k, v = c.data(1, 100)
    v = v.abs() + 1.0
    v[:, :, :, 1::2] *= -1
    c.append(1, 100, data=(k, v))
    page = int(c.gpu.table[0, 2])
    c.gpu.v_scale[page] = float("inf")
    q = torch.randn(1, 3, H, 64, generator=c.g).to(dtype).cuda()
    o = c.m.l1attn_paged(q, c.gpu)
    assert (o[..., 0::2] == float("inf")).all() and (o[..., 1::2] == -float("inf")).all()


@pytest.mark.parametrize("H", [2, 12])
def test_two_calls_at_once(H):
    c = Pair(N=80, P=32, Hk=2, W=64, Wv=64, rows=4, M=40, seed=4)
    c.append(4, 600, counts=[600, 550, 3, 0])
    qs = [torch.randn(4, 2, H, 64, generator=c.g).to(BF16).cuda() for _ in range(2)]
    want = [c.m.l1attn_paged(q, c.gpu) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(4):
        got = []
        for q, s in zip(qs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(c.m.l1attn_paged(q, c.gpu))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H", [2, 12])
def test_a_pool_that_the_caller_filled(H, dtype):
    # every code there is, and scales of either sign
    c = Pair(N=30, P=16, Hk=2, W=64, Wv=64, rows=2, M=10, dtype=dtype, seed=8)
    c.append(2, 150, counts=[150, 20])
    for to, codes in ((c.gpu.k_pages, c.plain.pages[0]), (c.gpu.v_pages, c.plain.pages[1])):
        codes.copy_(torch.randint(-128, 128, codes.shape, generator=c.g).to(torch.int8))
        to.copy_(codes)
    for to, scale in ((c.gpu.k_scale, c.plain.scale[0]), (c.gpu.v_scale, c.plain.scale[1])):
        scale.copy_((torch.rand(scale.shape, generator=c.g) - 0.5) / 64)
        to.copy_(scale)
    c.attend(2, 2, H)


@pytest.mark.parametrize("new", [0.01, 3.0, 100.0])
def test_append_to_a_pool_that_the_caller_filled(new):
    # scales of either sign: what the old tokens are stays, to half a step of the page's new scale and its float32 roundings (to a
    # whole step for the code -128, which has no opposite), and so do the new ones
    c = Pair(N=30, P=16, Hk=2, W=64, Wv=64, rows=2, M=10, dtype=F32, seed=8)
    c.append(2, 150, counts=[150, 20])
    for x in (c.gpu.k_pages, c.gpu.v_pages):
        x.copy_(torch.randint(-128, 128, x.shape, generator=c.g).to(torch.int8))
    for x in (c.gpu.k_scale, c.gpu.v_scale):
        x.copy_((torch.rand(x.shape, generator=c.g) - 0.5) / 16)

    def last_page(row, place):
        page = int(c.gpu.table[row, place // 16])
        return [(codes[page].cpu(), scale[page].double().cpu()[:, None, None]) for codes, scale in ((c.gpu.k_pages, c.gpu.k_scale), (c.gpu.v_pages, c.gpu.v_scale))]
    before = [last_page(row, n) for row, n in ((0, 150), (1, 20))]
    kv = c.data(2, 3, new)
    assert c.gpu.append(kv[0].cuda(), kv[1].cuda()).all()
    for row, n in ((0, 150), (1, 20)):
        at = n % 16
        for (was, old), (now, scale), x in zip(before[row], last_page(row, n), kv):
            assert (scale >= old.abs()).all()
            step = scale * (1 + 2.0 ** -15)
            room = torch.where(was == -128, step, step / 2)
            assert ((now * scale - was * old)[:, :at].abs() <= room[:, :at]).all()
            assert ((now * scale)[:, at:at + 3] - x[row].double().transpose(0, 1)).abs().le(step / 2).all()


def test_pages_that_are_not_there_give_no_tokens():
    c = Pair(N=40, rows=2, M=8)
    c.append(2, 100)
    o = c.attend(1, 1, 2)
    # a table that someone has damaged: the tokens of such pages are left out, nothing else is read
    c.gpu.table[1, 2], c.gpu.table[1, 4] = 40, -7
    q = torch.randn(2, 1, 2, 32).to(BF16).cuda()
    a = c.m.l1attn_paged(q, c.gpu)
    keep = torch.ones(100, dtype=torch.bool)
    keep[32:48] = keep[64:80] = False
    k, v = c.plain.tokens(1)
    for h in range(2):
        x = torch.exp(-(q[1, 0, h].double().cpu() - k[keep, h]).abs().sum(1) / 32 ** 0.5)
        want = (x / (1 + x.sum())) @ v[keep, h]
        assert (a[1, 0, h].double().cpu() - want).abs().max() <= 2.0 ** -8 * (v.abs().max())
    assert torch.isfinite(o).all()


def test_a_run_of_serving_calls_matches_the_training_operator():
    # prompt, steps, a drafted token that is rejected, a fork: as the masked operator on the cache's values sees it
    import l1attn_masked_cuda as mm
    c = Pair(N=60, P=32, Hk=2, W=64, Wv=64, rows=3, M=10, dtype=F32)
    c.append(2, 90, counts=[90, 41])
    for step in range(3):
        c.append(2, 1)
    c.append(2, 4)
    c.free([0, 1], keep=[93, 44])
    c.fork([0], [2])
    c.append(3, 2)
    c.compact()
    g = torch.Generator().manual_seed(1)
    for s in range(3):
        k, v = (x.float().cuda()[None] for x in c.plain.tokens(s))
        q = torch.randn(1, 2, 4, 64, generator=g).cuda()
        o = c.m.L1AttnPaged(softcap=9.0, slopes=(0.5, 0.1, 0.0, 0.2))(q, c.gpu, seqs=c.ints([s]))
        with torch.no_grad():
            want = mm.L1AttnMasked(softcap=9.0, slopes=(0.5, 0.1, 0.0, 0.2))(q, k, v)
        # both in float32: see lm_forms for the bound of either
        assert (o - want).abs().max() <= 2 * 2.0 ** -24 * (3 * 64 + 64 + 1) * v.abs().max()


def test_slopes_as_tensors_that_change_in_place():
    c = Pair(rows=1)
    c.append(1, 60)
    q = torch.randn(1, 1, 2, 32, generator=c.g).to(BF16).cuda()
    slopes = (torch.tensor(0.5), torch.tensor(0.25))
    for x in (0.5, 3.0):
        slopes[0].fill_(x)
        want = c.m.l1attn_paged(q, c.gpu, slopes=[x, 0.25])
        assert torch.equal(c.m.l1attn_paged(q, c.gpu, slopes=slopes), want)
        assert torch.equal(c.m.l1attn_paged(q, c.gpu, slopes=torch.stack(slopes)), want)


def test_graph_of_a_decode_step_and_other_streams():
    import l1attn_paged_cuda as m

    def fresh():
        c = m.L1PagedCache.empty(64, 16, 2, 32, 4, 12, device="cuda")
        g = torch.Generator().manual_seed(3)
        k, v = (torch.randn(4, 45, 2, 32, generator=g).to(BF16).cuda() for _ in range(2))
        assert c.append(k, v).all()
        return c
    state = lambda c: [x.clone() for x in (c.table, c.lens, c.refs, c.n_free, c.k_pages, c.v_pages, c.k_scale, c.v_scale)]  # noqa: E731
    k, v = (torch.zeros(4, 1, 2, 32, dtype=BF16, device="cuda") for _ in range(2))
    q = torch.zeros(4, 1, 4, 32, dtype=BF16, device="cuda")

    def step(c):
        served = c.append(k, v)
        return served, m.l1attn_paged(q, c, slopes=(0.1, 0.2, 0.3, 0.4))
    eager, captured, other = fresh(), fresh(), fresh()
    step(fresh())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured)
    s = torch.cuda.Stream()
    for i in range(6):
        g = torch.Generator().manual_seed(10 + i)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        want = step(eager)
        graph.replay()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step(other)
        torch.cuda.synchronize()
        for a in (out, got):
            assert all(torch.equal(x, y) for x, y in zip(a, want))
        for c in (captured, other):
            assert all(torch.equal(x, y) for x, y in zip(state(c), state(eager)))


def test_compact_with_a_table_of_more_than_2_32_entries():
    import l1attn_paged_cuda as m
    M = 1 << 24
    N, rows = 8, 260
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    table = torch.full((rows, M), -1, dtype=torch.int32, device="cuda")
    c = m.L1PagedCache(z(N, 1, 16, 16, dtype=torch.int8), z(N, 1, 16, 16, dtype=torch.int8), z(N, 1, dtype=F32), z(N, 1, dtype=F32), table, z(rows), z(N),
                       torch.arange(N - 1, -1, -1, dtype=torch.int32, device="cuda"), z(1) + N)
    x = torch.randn(2, 20, 1, 16, generator=torch.Generator().manual_seed(1)).cuda()
    assert c.append(x, x, seqs=torch.tensor([3, 259], dtype=torch.int32, device="cuda")).all()  # pages 0, 1 and 2, 3
    q = x[:, -1:].contiguous()
    seqs = torch.tensor([259], dtype=torch.int32, device="cuda")
    want = m.l1attn_paged(q[1:], c, seqs=seqs)
    c.free(torch.tensor([3], dtype=torch.int32, device="cuda"))
    assert int(c.compact()) == 2 and table[259, :3].tolist() == [0, 1, -1]
    assert torch.equal(m.l1attn_paged(q[1:], c, seqs=seqs), want)


def test_random_walk():
    import random
    r = random.Random(5)
    c = Pair(N=50, P=16, Hk=2, W=20, Wv=36, rows=7, M=6, seed=9)
    for step in range(60):
        what = r.choice(("append", "append", "append", "fork", "free", "compact"))
        seqs = r.sample(range(7), r.randint(1, 7))
        if what == "append":
            n = r.choice((1, 2, 17, 40))
            c.append(len(seqs), n, seqs=seqs, counts=[r.randint(0, n) for _ in seqs], scale=r.choice((0.1, 1.0, 4.0)))
        elif what == "fork":
            c.fork([r.randrange(7) for _ in seqs], seqs)
        elif what == "free":
            c.free(seqs, keep=r.choice((None, [r.randint(0, 90) for _ in seqs])))
        else:
            c.compact()
        if step % 6 == 0:
            c.attend(7, 1, 2)
