"""Bounds of pages, the choice of pages by them, and attention over chosen pages (csrc/kernels/paged_select.hip,
attention_paged*.hip) against their definitions in 64 bits."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests.gpu_util import call, host, ptr, stream  # noqa: E402
from tests.paged_codes_ref import Cache, bounds, select  # noqa: E402
from tests.paged_ref import CODE, HALF, TORCH  # noqa: E402
from tests.test_gpu_attn_paged import Call  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


CACHES = ["f32", "bf16", "e4m3", "e2m1"]
TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "e4m3"), ("bf16", "e2m1"), ("f32", "e4m3"), ("f32", "e2m1")]


def _bound_type(cache):
    return torch.float32 if cache == "f32" else torch.bfloat16


def _run_bounds(p, out):
    c = p.struct()
    T = p.offs[-1] + 3
    call("aic_hip_kv_bounds", c, ptr(out), ptr(p.dev_offs), ptr(p.dev_lens), p.B, T, stream())


# ------------------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("ns,lens,Hkv,hd,ps,first", [([1], [1], 1, 32, 1, 0), ([1, 1, 1], [5, 16, 17], 3, 64, 16, 0),
                                                     ([7, 0, 300, 1], [9, 4, 300, 64], 2, 128, 24, 0), ([40, 3], [33, 2], 4, 128, 7, 2),
                                                     ([0, 0, 5, 0], [0, 3, 5, 0], 1, 64, 128, 0), ([33] * 9 + [1] * 80, [40] * 9 + [70] * 80, 2, 32, 64, 1)])
def test_bounds(cache, ns, lens, Hkv, hd, ps, first):
    p = Cache(ns, lens, Hkv, hd, ps, cache, seed=hd + ps, first=first)
    out = torch.full((p.n_pages, Hkv, 2, hd), 7.0, dtype=_bound_type(cache), device="cuda")
    want = bounds(p, out.double().cpu().numpy())
    _run_bounds(p, out)
    assert np.array_equal(out.double().cpu().numpy(), want)


@pytest.mark.parametrize("cache", CACHES)
def test_bounds_of_what_is_no_number_or_no_page(cache):
    """NaN inside and behind the filled part; pages outside the pool and past the table."""
    p = Cache([20, 9, 4], [30, 9, 70], 2, 64, 8, cache, seed=5, extra_table=0)
    t = p.pool["k"][0 if cache != "e2m1" else 1]
    nan = float("nan") if cache in ("f32", "bf16") else 0x7f if cache == "e4m3" else 255
    for b, pos in ((0, 12), (1, 3)):
        page, slot = p.place(b, pos)
        t[page, 1, slot, 0] = nan
        p.k[page, 1, slot, :32 if cache == "e2m1" else 1] = np.nan
    page, slot = p.place(0, 29)
    t[page, :, slot + 1:] = nan      # behind the sequence
    p.table[2, 8] = p.n_pages        # positions 64 .. 71
    out = torch.full((p.n_pages, 2, 2, 64), 7.0, dtype=_bound_type(cache), device="cuda")
    want = bounds(p, out.double().cpu().numpy())
    assert np.isnan(want).any()
    _run_bounds(p, out)
    assert np.array_equal(out.double().cpu().numpy(), want, equal_nan=True)


# -------------------------------------------------------------------------------------- choice
class Choice:
    def __init__(self, p, H, dt, first=1, last=2, n_sel=8, pad=0, shift=0, tail=3, seed=0, tied=False, max_len=None):
        self.p, self.H, self.dt, self.cut = p, H, dt, (first, last, n_sel)
        self.T, self.w = p.offs[-1] + tail, H * p.hd
        self.ld = self.w + pad
        rng = np.random.default_rng(seed)
        q = rng.standard_normal((self.T, self.ld))
        mid, reach = rng.standard_normal((2, p.n_pages, p.Hkv, p.hd))
        if tied:  # whole numbers of few values: many equal scores
            q, mid, reach = np.sign(q), np.round(mid), np.ones_like(reach)
        buf = torch.empty(self.T * self.ld + shift, dtype=TORCH[dt], device="cuda")
        self.q = buf[shift:].view(self.T, self.ld)
        self.q.copy_(torch.from_numpy(q))
        self.bounds = torch.from_numpy(np.stack([mid - abs(reach), mid + abs(reach)], 2)).to(_bound_type(p.cache)).cuda()
        self.max_len = max(max(p.lens), 0) if max_len is None else max_len
        self.picked = torch.full((self.T, p.Hkv, n_sel), 77, dtype=torch.int32, device="cuda")
        self.lens = torch.full((self.T, p.Hkv), 77, dtype=torch.int64, device="cuda")

    def args(self, ws=None, max_q=None):
        p = self.p
        c = p.struct()
        return (c, ptr(self.bounds), ptr(self.q), self.ld, ptr(p.dev_offs), ptr(p.dev_lens), p.B, self.T, max(p.ns) if max_q is None else max_q,
                self.max_len, self.H, *self.cut, ptr(self.picked), ptr(self.lens), *((None, 0) if ws is None else (ptr(ws), ws.numel())),
                CODE[self.dt])

    def bytes(self):
        return _lib.load().aic_hip_kv_select_workspace(self.p.struct(), self.T, self.max_len)

    def want(self):
        q = self.q[:, :self.w].double().cpu().numpy().reshape(self.T, self.H, self.p.hd)
        return select(self.p, self.bounds.double().cpu().numpy(), q, self.H, *self.cut, self.max_len)

    def run(self, ws=None, max_q=None):
        call("aic_hip_kv_select", *self.args(ws, max_q), stream())
        return self

    def check(self):
        picked, lens = self.want()
        assert np.array_equal(host(self.lens), lens)
        assert np.array_equal(host(self.picked), picked)
        return self


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens,H,Hkv,hd,ps,first,last,n_sel", [
    ([1], [1], 1, 1, 32, 1, 0, 1, 1), ([1], [100], 2, 1, 32, 1, 0, 1, 1), ([1, 1, 1], [500, 16, 17], 6, 3, 64, 16, 1, 2, 8),
    ([7, 0, 30, 1], [900, 4, 300, 64], 4, 2, 128, 24, 2, 1, 5), ([40, 3], [33, 2], 4, 4, 128, 7, 0, 1, 3),
    ([0, 0, 5, 0], [0, 3, 700, 0], 3, 1, 64, 4, 3, 3, 6), ([9, 2], [2000, 3000], 40, 1, 64, 16, 1, 2, 33),
    ([3] * 70, [400] * 70, 4, 2, 32, 8, 1, 1, 16), ([1], [6000], 8, 1, 128, 2, 1, 2, 300), ([33], [600], 16, 16, 64, 16, 1, 2, 8)])
def test_choice(dt, cache, ns, lens, H, Hkv, hd, ps, first, last, n_sel):
    p = Cache(ns, lens, Hkv, hd, ps, cache, seed=hd)
    Choice(p, H, dt, first, last, n_sel, pad=hd % 5, shift=len(ns) % 2).run().check()


@pytest.mark.parametrize("n_sel", [3, 4, 20, 100, 254])
@pytest.mark.parametrize("H", [1, 4])
def test_equal_scores(n_sel, H):
    """Many pages of one score: the lower positions."""
    p = Cache([2, 1], [1020, 700], 1, 32, 4, "bf16", seed=n_sel)
    Choice(p, H, "bf16", 1, 2, n_sel, tied=True).run().check()
    a = Choice(p, H, "bf16", 1, 2, n_sel)
    a.bounds.fill_(1.0)  # all pages alike
    a.run().check()


def test_scores_of_both_signs_and_sizes():
    p = Cache([4], [2000], 2, 64, 8, "f32", seed=1)
    a = Choice(p, 4, "f32", 0, 1, 17)
    scale = torch.from_numpy(10.0 ** np.random.default_rng(2).integers(-30, 30, (p.n_pages, 1, 1, 1))).cuda()
    a.bounds = (a.bounds.double() * scale).float()
    a.q[1] = 0     # every score is 0, of either sign
    a.q[2] *= -1e30
    a.run().check()


def test_what_is_no_number():
    """NaN and infinities in bounds and queries, and pages that are none."""
    p = Cache([3, 2], [900, 300], 1, 32, 8, "bf16", seed=1, extra_table=0)
    p.table[0, 20] = -1
    p.table[0, 33] = p.n_pages
    p.table[1, 7] = 2 ** 31 - 1
    a = Choice(p, 2, "bf16", 1, 2, 9)
    a.bounds[p.table[0, 50], 0, 1, 3] = float("nan")
    a.bounds[p.table[0, 60], 0] = float("-inf")
    a.bounds[p.table[0, 70], 0, 1] = float("inf")
    a.bounds[p.table[1, 11], 0, 0] = float("nan")
    a.q[1, 5] = float("nan")
    a.q[2, 40] = float("inf")
    a.run().check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("ns,lens,H,Hkv,hd,n_sel", [([37, 0, 1, 64], [900, 5, 300, 700], 8, 2, 128, 9), ([100], [800], 20, 1, 64, 12),
                                                    ([2] * 9, [1100] * 9, 24, 2, 32, 5), ([5, 3], [3000, 2000], 40, 1, 128, 20)])
def test_choice_of_many_rows(dt, ns, lens, H, Hkv, hd, n_sel):
    """Chunks, large groups and groups of more than 32 heads; a page with infinities among the others."""
    p = Cache(ns, lens, Hkv, hd, 16, dt, seed=hd)
    a = Choice(p, H, dt, 1, 2, n_sel, pad=8, tied=hd == 32)
    a.run().check()
    a.bounds[p.table[0, 10], :, 1, 5] = float("inf")
    a.bounds[p.table[0, 20], 0, 0, 7] = float("-inf")
    a.bounds[p.table[0, 21], 0, :, 8] = float("nan")
    a.q[0, 7], a.q[1, 5] = 0.0, -0.0
    a.run().check()


@pytest.mark.parametrize("H", [2, 16])
def test_zeros_of_either_sign_beside_infinities(H):
    """An element of q that is 0 or -0 meets the page's greatest."""
    p = Cache([3], [900], 1, 32, 8, "bf16", seed=1)
    a = Choice(p, H, "bf16", 1, 2, 9)
    a.q[0, 3], a.q[1, 3], a.q[1, 35], a.q[2, 35] = 0.0, -0.0, -0.0, 0.0
    a.bounds[p.table[0, 30], 0, 0, 3] = float("-inf")
    a.bounds[p.table[0, 60], 0, 1, 3] = float("inf")
    a.run().check()


@pytest.mark.parametrize("max_len", [1, 100, 333])
def test_longer_than_promised(max_len):
    """Rows past max_len get a page that is none; the others are right, and nothing is written past the workspace."""
    p = Cache([4, 1, 90], [900, 300, 370], 2, 64, 16, "bf16", seed=9)
    a = Choice(p, 4, "bf16", 1, 2, 6, max_len=max_len)
    n = a.bytes()
    ws = torch.full((n + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    c = a.args(ws[:max(n, 16)] if n % 16 == 0 else ws, max_q=1)
    call("aic_hip_kv_select", *c, stream())
    a.check()
    assert (ws[n:] == 0x5a).all()


def test_rows_before_the_first_and_none():
    p = Cache([0, 2, 0], [0, 90, 5], 2, 32, 4, "bf16", seed=1, first=3)
    Choice(p, 2, "bf16", 1, 1, 4).run().check()
    p = Cache([0, 0], [0, 9], 2, 32, 4, "bf16", seed=1)
    a = Choice(p, 2, "bf16", 1, 1, 4).run()
    assert (a.picked == -1).all() and (a.lens == -1).all()


def test_choice_captured():
    p = Cache([2, 1], [3000, 700], 2, 64, 16, "bf16", seed=4)
    a = Choice(p, 8, "bf16", 1, 2, 16)
    ws = torch.empty(a.bytes(), dtype=torch.uint8, device="cuda")
    args = a.args(ws)
    held = p.dev_table, p.dev_offs, p.dev_lens  # the graph's, while later calls make their own
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call("aic_hip_kv_select", *args, torch.cuda.current_stream().cuda_stream)
        with pytest.raises(_lib.AicError, match="captured"):
            call("aic_hip_kv_select", *args[:-3], None, 0, args[-1], torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        a.q.copy_(torch.randn_like(a.q.float()) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        a.check()
        Choice(p, 8, "bf16", 1, 2, 16).run().check()
    del held


# ---------------------------------------------------------------------------- attention over them
def attention(p, q, H, picked, lens, scale):
    """(o, lse, sum of weighed |v|, bound of a score's error) in 64 bits."""
    T, G = q.shape[0], H // p.Hkv
    o, lse = np.full((T, H, p.hd), np.nan), np.full((T, H), np.nan)
    ab, sb = np.zeros((T, H, p.hd)), np.zeros((T, H))
    for t in range(T):
        for h in range(p.Hkv):
            n = int(lens[t, h])
            if n < 0:
                continue
            j = np.arange(n)
            if n == 0:
                o[t, h * G:(h + 1) * G], lse[t, h * G:(h + 1) * G] = 0, -np.inf
                continue
            pages = np.array([picked[t, h, i] if i < picked.shape[2] else -1 for i in j // p.ps])
            ok = (pages >= 0) & (pages < p.n_pages)
            K, V = (np.where(ok[:, None], getattr(p, x)[np.where(ok, pages, 0), h, j % p.ps], np.nan) for x in "kv")
            x = q[t, h * G:(h + 1) * G]
            with np.errstate(all="ignore"):
                s = scale * (x @ K.T)
                m = s.max(1, keepdims=True)
                w = np.exp(s - m)
                tot = w.sum(1, keepdims=True)
                o[t, h * G:(h + 1) * G], ab[t, h * G:(h + 1) * G] = (w / tot) @ V, (w / tot) @ np.abs(V)
                lse[t, h * G:(h + 1) * G] = (m + np.log(tot))[:, 0]
                sb[t, h * G:(h + 1) * G] = scale * (np.abs(x) @ np.abs(K.T)).max(1) * (p.hd + 2) * 2.0 ** -24
    return o, lse, ab, sb


class Picked:
    """A call over given pages; the tolerances of tests/paged_ref.py's check_attention."""

    def __init__(self, p, H, dt, picked, lens, pad=0, shift=0, seed=0, with_lse=True):
        self.p, self.H, self.dt, self.scale = p, H, dt, 1.0 / math.sqrt(p.hd)
        self.picked, self.lens = np.ascontiguousarray(picked, np.int32), np.ascontiguousarray(lens, np.int64)
        self.T, self.w = self.lens.shape[0], H * p.hd
        self.ld, self.shift = self.w + pad, shift
        rng = np.random.default_rng(seed + 2)
        self.q = torch.empty(self.T * self.ld + shift, dtype=TORCH[dt], device="cuda")[shift:].view(self.T, self.ld)
        self.q.copy_(torch.from_numpy(rng.standard_normal((self.T, self.ld))))
        self.o = torch.full((self.T * self.ld + shift,), 7.0, dtype=TORCH[dt], device="cuda")[shift:].view(self.T, self.ld)
        self.lse = torch.full((self.T, H), 7.0, device="cuda") if with_lse else None
        self.dev = torch.from_numpy(self.picked).cuda(), torch.from_numpy(self.lens).cuda()

    def bytes(self):
        return _lib.load().aic_hip_attn_paged_selected_workspace(self.p.struct(), self.T, self.picked.shape[2], self.H)

    def args(self, ws=None):
        c = self.p.struct()
        return (c, ptr(self.q), self.ld, ptr(self.o), self.ld, ptr(self.lse), ptr(self.dev[0]), ptr(self.dev[1]), self.T,
                self.picked.shape[2], self.H, self.scale, *((None, 0) if ws is None else (ptr(ws), ws.numel())), CODE[self.dt])

    def run(self, ws=None):
        call("aic_hip_attn_paged_selected", *self.args(ws), stream())
        return self

    def check(self):
        p, dt = self.p, self.dt
        q = self.q[:, :self.w].double().cpu().numpy().reshape(self.T, self.H, p.hd)
        o, l, ab, sb = attention(p, q, self.H, self.picked, self.lens, self.scale)
        left = np.repeat(self.lens < 0, self.H // p.Hkv, 1)
        g = host(self.o.contiguous())[:, :self.w].reshape(self.T, self.H, p.hd).astype(np.float64)
        assert (g[left] == 7.0).all() and (host(self.o)[:, self.w:] == 7.0).all()
        g, r, ab, sb = g[~left], o[~left], ab[~left], sb[~left]
        assert np.array_equal(np.isnan(g), np.isnan(r))
        fine = np.isfinite(r)
        tol = (4 * sb[..., None] + 2.0 ** -18) * ab + 2 ** -40
        tol = tol + HALF[dt] * np.abs(r) * 1.01 + (HALF["bf16"] * ab * 1.01 if dt == "bf16" else 0)
        assert (np.abs(g - r)[fine] <= tol[fine]).all(), float((np.abs(g - r) / tol)[fine].max())
        if self.lse is not None:
            a, e = host(self.lse).astype(np.float64), l
            assert (a[left] == 7.0).all()
            a, e = a[~left], e[~left]
            assert np.array_equal(np.isnan(a), np.isnan(e))
            fine = np.isfinite(e)
            assert np.array_equal(a[~fine & ~np.isnan(e)], e[~fine & ~np.isnan(e)])
            assert (np.abs(a[fine] - e[fine]) <= 2 * sb[fine] + 2.0 ** -17 + 2.0 ** -22 * np.abs(e[fine])).all()
        return self


def _random_pages(p, T, n_sel, seed):
    """Pages in any order, lengths from none to all of them; some rows are nobody's."""
    rng = np.random.default_rng(seed)
    picked = np.stack([rng.permutation(p.n_pages)[:n_sel] for _ in range(T * p.Hkv)]).reshape(T, p.Hkv, n_sel)
    lens = rng.integers(0, n_sel * p.ps + 1, (T, p.Hkv))
    lens[0, 0] = n_sel * p.ps
    if T > 2:
        lens[1] = -1
        lens[2, p.Hkv - 1] = 0
    return picked, lens


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("T,H,Hkv,hd,ps,n_sel,pad,shift", [
    (1, 1, 1, 32, 1, 1, 0, 0), (1, 16, 2, 128, 64, 32, 0, 0), (7, 12, 12, 64, 16, 9, 8, 0), (5, 8, 1, 128, 24, 11, 0, 0),
    (40, 4, 2, 32, 7, 20, 3, 1), (3, 40, 1, 64, 16, 33, 0, 0), (4, 6, 2, 128, 16, 100, 0, 0), (130, 2, 1, 64, 32, 5, 0, 0)])
def test_attention_over_chosen_pages(dt, cache, T, H, Hkv, hd, ps, n_sel, pad, shift):
    p = Cache([1], [ps * (n_sel + 3)], Hkv, hd, ps, cache, seed=hd + T)
    Picked(p, H, dt, *_random_pages(p, T, n_sel, T), pad=pad, shift=shift).run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("T,H,Hkv,hd,n_sel", [(1, 4, 1, 64, 200), (2, 16, 2, 128, 150), (3, 3, 3, 32, 130), (2, 5, 1, 64, 100)])
def test_chosen_pages_split_among_blocks(dt, cache, T, H, Hkv, hd, n_sel):
    p = Cache([1], [16 * n_sel], Hkv, hd, 16, cache, seed=hd)
    at = _random_pages(p, T, n_sel, T)
    a = Picked(p, H, dt, *at)
    assert a.bytes() > 0
    a.run(torch.full((a.bytes(),), 0xff, dtype=torch.uint8, device="cuda")).check()
    b = Picked(p, H, dt, *at, with_lse=False).run().check()
    assert torch.equal(a.o, b.o)
    with pytest.raises(_lib.AicError, match="workspace"):
        Picked(p, H, dt, *at).run(torch.empty(a.bytes() - 16, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("T,H,Hkv,hd", [(17, 8, 8, 64), (30, 16, 8, 32), (38, 8, 8, 64), (75, 16, 8, 32)])
def test_chosen_pages_of_many_rows(dt, cache, T, H, Hkv, hd):
    """A block for each row and head, and blocks that share more rows than they have threads."""
    p = Cache([1], [16 * 110], Hkv, hd, 16, cache, seed=T)
    Picked(p, H, dt, *_random_pages(p, T, 105, T)).run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
def test_chosen_pages_that_are_none(dt, cache):
    p = Cache([1], [400], 2, 64, 16, cache, seed=3)
    picked, lens = _random_pages(p, 6, 10, 1)
    picked[0, 0, 3] = -1
    picked[3, 1, 0] = p.n_pages
    picked[4, 0, 9] = 2 ** 31 - 1
    lens[3], lens[4] = 100, 100          # the last of row 4's pages is not reached
    lens[5, 1] = 161                     # one position past its pages
    Picked(p, 4, dt, picked, lens).run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("T,n_sel", [(4, 10), (3, 90), (130, 80)])
def test_lengths_past_the_pages(dt, cache, T, n_sel):
    """However large: NaN, as one position past them; the other rows as they are."""
    p = Cache([1], [16 * (n_sel + 2)], 2, 32, 16, cache, seed=3)
    picked, lens = _random_pages(p, T, n_sel, 1)
    want = Picked(p, 4, dt, picked, lens).run().o.clone().view(T, 2, 64)
    lens[1, 0], lens[2, 1] = 2 ** 31, 2 ** 62
    got = Picked(p, 4, dt, picked, lens).run().o.view(T, 2, 64)
    past = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    past[1, 0] = past[2, 1] = True
    assert torch.isnan(got[past]).all() and torch.equal(got[~past], want[~past])


def test_two_streams_at_once():
    """Choices and attention on two streams, with the streams' own scratch memory, as one after the other."""
    calls, want = [], []
    for seed in range(2):
        p = Cache([3, 1], [5000, 3000], 2, 64, 16, "bf16", seed=seed)
        a = Choice(p, 8, "bf16", 1, 2, 100, seed=seed)
        a.run()
        b = Picked(p, 8, "bf16", host(a.picked), host(a.lens), seed=seed).run()
        want.append((a.picked.clone(), b.o.clone()))
        calls.append((a, b, a.args(), (p.dev_table, p.dev_offs, p.dev_lens), b.args(), (p.dev_table, p.dev_offs, p.dev_lens)))
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        for a, b, *_rest in calls:
            a.picked.zero_(), b.o.fill_(7.0)  # rows of nobody stay
        torch.cuda.synchronize()
        for _ in range(3):
            for s, (a, b, c, _c, d, _d) in zip(streams, calls):
                call("aic_hip_kv_select", *c, s.cuda_stream)
                call("aic_hip_attn_paged_selected", *d, s.cuda_stream)
        torch.cuda.synchronize()
        for (a, b, *_rest), (picked, o) in zip(calls, want):
            assert torch.equal(a.picked, picked) and torch.equal(b.o, o)


@pytest.mark.parametrize("dt,cache", [("bf16", "e2m1"), ("bf16", "bf16"), ("f32", "f32")])
def test_chosen_pages_captured(dt, cache):
    p = Cache([1], [4000], 2, 64, 16, cache, seed=5)
    at = _random_pages(p, 3, 120, 2)
    for own in (True, False):
        a = Picked(p, 8, dt, *at)
        ws = torch.empty(max(a.bytes(), 16), dtype=torch.uint8, device="cuda") if own else None
        args = a.args(ws)
        held = p.dev_table, p.dev_offs, p.dev_lens  # the graph's, while later calls make their own
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call("aic_hip_attn_paged_selected", *args, torch.cuda.current_stream().cuda_stream)
        for _ in range(3):
            a.o.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            a.check()
            Picked(p, 8, dt, *at).run()
        del held


# ---------------------------------------------------------------------------------- all together
@pytest.mark.parametrize("dt,cache", TYPES)
def test_serving_a_growing_cache(dt, cache):
    """Prompts, then tokens: appended with their rotation, bounds brought up to date, pages chosen, attended over.  The bounds
    hold every cached key; the choice is the definition's for them; attention is the definition's over the choice, and
    attn_paged's where the choice is everything."""
    H, Hkv, hd, ps, n_sel, B = 4, 2, 64, 8, 5, 3
    steps = [[30, 9, 1], [1, 1, 1], [3, 1, 2], [17, 1, 9], [1, 1, 1]]
    total = [sum(s[b] for s in steps) for b in range(B)]
    p = Cache([1] * B, total, Hkv, hd, ps, cache, seed=1)
    for name in "kv":
        for t in p.pool[name]:
            if t is not None:
                t.view(torch.uint8).fill_(0xff)
    bound = torch.full((p.n_pages, Hkv, 2, hd), float("nan"), dtype=_bound_type(cache), device="cuda")
    c, s = (np.empty((max(total), hd // 2), np.float32) for _ in range(2))
    call("aic_hip_rope_tables", c.ctypes.data, s.ctypes.data, max(total), hd, 10000.0)
    c, s = torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    done = [0] * B
    for ns in steps:
        done = [a + n for a, n in zip(done, ns)]
        p.ns, p.lens, p.offs = list(ns), list(done), [sum(ns[:b]) for b in range(B + 1)]
        T, w = p.offs[-1], H * hd
        x = torch.randn((T, (H + 2 * Hkv) * hd), generator=g, device="cuda").to(TORCH[dt])
        size, ld = x.element_size(), x.shape[1]
        desc = p.struct()
        alive = p.dev_table, p.dev_offs, p.dev_lens  # while later calls make their own
        batch = (*(ptr(t) for t in alive[1:]), B, T)
        call("aic_hip_kv_append", desc, ptr(x), ld, ptr(x), ld, H, ptr(x) + w * size, ptr(x) + (w + Hkv * hd) * size, ld, ptr(c), ptr(s),
             c.shape[0], *batch, CODE[dt], stream())
        call("aic_hip_kv_bounds", desc, ptr(bound), *batch, stream())
        # what the cache holds now
        n = max(done)
        one = torch.tensor([sum(done[:b]) for b in range(B + 1)], device="cuda")
        k, v = (torch.empty((sum(done), Hkv * hd), dtype=TORCH[dt], device="cuda") for _ in range(2))
        call("aic_hip_kv_read", desc, ptr(k), ptr(v), Hkv * hd, ptr(one), ptr(alive[2]), B, sum(done), CODE[dt], stream())
        for name, rows in (("k", k), ("v", v)):
            held = np.full(getattr(p, name).shape, np.nan)
            rows = rows.double().cpu().numpy().reshape(-1, Hkv, hd)
            for b in range(B):
                for j in range(done[b]):
                    page, slot = p.place(b, j)
                    held[page, :, slot] = rows[sum(done[:b]) + j]
            setattr(p, name, held)
        lo, hi = (bound[:, :, i].double().cpu().numpy() for i in range(2))
        for b in range(B):
            for j in range(done[b]):
                page, slot = p.place(b, j)
                assert (lo[page] <= p.k[page, :, slot]).all() and (p.k[page, :, slot] <= hi[page]).all()
        q = x[:, :w].double().cpu().numpy().reshape(T, H, hd)
        for sel in (n_sel, -(-n // ps)):
            picked = torch.empty((T, Hkv, sel), dtype=torch.int32, device="cuda")
            lens = torch.empty((T, Hkv), dtype=torch.int64, device="cuda")
            call("aic_hip_kv_select", desc, ptr(bound), ptr(x), ld, *batch, max(ns), n, H, 1, 2, sel, ptr(picked), ptr(lens), None, 0,
                 CODE[dt], stream())
            want = select(p, np.stack([lo, hi], 2), q, H, 1, 2, sel, n)
            assert np.array_equal(host(picked), want[0]) and np.array_equal(host(lens), want[1])
            a = Picked(p, H, dt, *want)
            a.q = x
            a.ld = ld
            a.o = torch.full((T, ld), 7.0, dtype=TORCH[dt], device="cuda")
            a.dev = picked, lens
            a.run().check()
            if sel >= -(-n // ps):
                d = Call(p, H, dt, tail=0, q=x[:, :w])
                d.run().check()
