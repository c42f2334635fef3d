"""Attention over the paged key/value cache (csrc/kernels/attention_paged.hip) against its definition in 64 bits, at
the sizes, masks and values where its tiles and splits can go wrong.  Bounds: tests/paged_ref.py."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests.gpu_util import call, host, ptr, stream  # noqa: E402
from tests.paged_ref import CODE, HALF, TORCH, Paged, attention, check_attention, e4m3_decode, e4m3_encode  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


class Call:
    """One batch's buffers: q and o rows of H * hd + pad elements, `shift` elements into their storage, with rows
    behind the last sequence."""

    def __init__(self, p, H, dt, window=0, pad=0, shift=0, tail=3, seed=0, with_lse=True, scale=None, q=None):
        self.p, self.H, self.dt, self.window = p, H, dt, window
        self.scale = 1.0 / math.sqrt(p.hd) if scale is None else scale
        self.T, self.w = p.offs[-1] + tail, H * p.hd
        self.ld = self.w + pad
        rng = np.random.default_rng(seed + 11)
        self.q = self._rows(shift)[1]
        self.q.copy_(torch.from_numpy(rng.standard_normal((self.T, self.ld))) if q is None else q)
        self.buf, self.o = self._rows(shift)
        self.shift = shift
        self.lse = torch.full((self.T, H), 7.0, device="cuda") if with_lse else None

    def _rows(self, shift):
        buf = torch.full((self.T * self.ld + shift + 16,), 7.0, dtype=TORCH[self.dt], device="cuda")
        return buf, buf[shift:shift + self.T * self.ld].view(self.T, self.ld)

    def sizes(self):
        p = self.p
        return p.B, self.T, max(p.ns, default=0), max(max(p.lens, default=0), 0)

    def run(self, workspace=None, st=None):
        p = self.p
        c = p.struct()
        ws = (None, 0) if workspace is None else (ptr(workspace), workspace.numel())
        call("aic_hip_attn_paged", c, ptr(self.q), self.ld, ptr(self.o), self.ld, ptr(self.lse), ptr(p.dev_offs), ptr(p.dev_lens),
             *self.sizes(), self.H, self.window, self.scale, *ws, CODE[self.dt], stream() if st is None else st)
        return self

    def bytes(self):
        B, T, n, L = self.sizes()
        return _lib.load().aic_hip_attn_paged_workspace(self.p.struct(), B, T, n, L, self.H)

    def check(self):
        p = self.p
        q = self.q[:, :self.w].double().cpu().numpy().reshape(self.T, self.H, p.hd)
        got = host(self.o.contiguous())[:, :self.w].reshape(self.T, self.H, p.hd)
        check_attention(got, None if self.lse is None else host(self.lse), p, q, self.H, self.window, self.scale, self.dt)
        inside = np.zeros(self.buf.numel(), bool)  # nothing else was written
        rows = inside[self.shift:self.shift + self.T * self.ld].reshape(self.T, self.ld)
        rows[p.offs[0]:p.offs[-1], :self.w] = True
        assert np.all(host(self.buf)[~inside] == 7.0)
        if self.lse is not None:
            assert np.all(host(self.lse)[p.offs[-1]:] == 7.0) and np.all(host(self.lse)[:p.offs[0]] == 7.0)
        return self


TYPES = [("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f32"), ("f32", "e4m3")]
# (ns, lens, H, Hkv, hd, page size, window, pad, shift)
CASES = [
    ([1], [1], 1, 1, 32, 16, 0, 0, 0),                                   # one token that sees itself
    ([1, 1, 1, 1], [1, 31, 64, 65], 4, 2, 64, 16, 0, 0, 0),              # single tokens around a tile's edge
    ([1] * 5, [700, 3, 0, 129, 400], 8, 1, 128, 24, 0, 8, 0),            # one key/value head, an empty cache: no row sees a key
    ([5, 3, 1], [5, 90, 300], 12, 12, 64, 16, 0, 0, 0),                  # drafted tokens
    ([33, 0, 70, 1], [40, 17, 70, 260], 8, 2, 64, 32, 0, 0, 0),          # chunks of prompts, a sequence without rows
    ([130], [515], 2, 2, 128, 64, 0, 0, 0),                              # more than one query tile
    ([9, 40], [4, 33], 4, 4, 32, 7, 0, 3, 1),                            # rows before position 0: nothing seen; odd strides
    ([50, 1, 9], [210, 333, 64], 4, 1, 64, 16, 20, 0, 0),                # a window inside a tile
    ([150], [150], 3, 1, 32, 1, 64, 0, 0),                               # pages of one slot, window of a tile
    ([1, 2], [900, 1200], 16, 2, 128, 128, 100, 0, 0),                   # decoding in a window
    ([64, 64], [64, 128], 16, 8, 128, 64, 1, 0, 0),                      # a window of one: o = v
]


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens,H,Hkv,hd,ps,window,pad,shift", CASES)
def test_attention_over_pages(dt, cache, ns, lens, H, Hkv, hd, ps, window, pad, shift):
    p = Paged(ns, lens, Hkv, hd, ps, cache, seed=hd + len(ns))
    Call(p, H, dt, window, pad, shift).run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens,H,Hkv,hd", [([1, 1, 1], [4100, 700, 1], 8, 2, 64), ([3, 8, 0], [2500, 1100, 900], 4, 4, 32),
                                              ([60, 1], [1500, 3000], 2, 1, 128)])
def test_keys_split_among_blocks(dt, cache, ns, lens, H, Hkv, hd):
    """Few rows over long caches: the split form with the call's own workspace and with the stream's, exactly alike, with and
    without lse."""
    p = Paged(ns, lens, Hkv, hd, 16, cache, seed=hd)
    a = Call(p, H, dt)
    assert a.bytes() > 0
    ws = torch.full((a.bytes(),), 0xff, dtype=torch.uint8, device="cuda")  # NaN in every place
    a.run(ws).check()
    b = Call(p, H, dt, with_lse=False).run().check()
    assert torch.equal(a.o, b.o)
    with pytest.raises(_lib.AicError, match="workspace"):
        Call(p, H, dt).run(ws[:a.bytes() - 16])


@pytest.mark.parametrize("window", [0, 5])
def test_larger_than_promised(window):
    """max_q and max_len below what offsets and lens hold: the same rows, from other kernels."""
    p = Paged([20, 1, 90], [900, 1300, 95], 2, 64, 16, "bf16", seed=9)
    a = Call(p, 4, "bf16", window)
    a.sizes = lambda: (p.B, a.T, 1, 64)
    a.run().check()


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("ns,lens,window", [([40], [100], 0), ([3], [700], 0), ([1], [45], 0), ([60], [200], 30), ([1], [2000], 70)])
def test_what_is_not_seen_does_not_reach_a_row(dt, cache, ns, lens, window):
    """NaN and infinities in keys and values: only the rows that see their position show them."""
    n, L = ns[0], lens[0]
    spots = [("k", L - n + n // 2, np.nan), ("v", L - n + n // 3, np.inf), ("v", L - 1, np.nan), ("v", L - n + n // 3, -np.inf)]
    if window:
        spots += [("v", max(0, L - n - window + 2), np.inf), ("v", max(0, L - n - window), np.nan)]
    for name, pos, value in spots:
        p = Paged(ns, lens, 1, 64, 16, cache, seed=L)
        row = np.random.default_rng(1).standard_normal(p.hd)
        row[5] = value
        p.set_row(name, 0, pos, 0, row)
        Call(p, 2, dt, window).run().check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_stale_values_behind_a_sequence(cache):
    """Slots past a sequence's length in its last page, and all pages of nobody, hold NaN."""
    p = Paged([1, 30, 2], [5, 37, 600], 2, 64, 64, cache, seed=2)
    used = np.zeros((p.n_pages, p.ps), bool)
    for b in range(p.B):
        for j in range(p.lens[b]):
            used[p.place(b, j)] = True
    free = torch.from_numpy(~used).cuda()
    for name in "kv":
        t = p.pool[name][0]
        t.view(torch.uint8).permute(0, 2, 1, 3)[free] = 0xff
    Call(p, 4, "bf16").run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
def test_pages_outside_the_pool(dt, cache):
    """Rows that see a position whose page id is out of range, or past the table's row, are NaN; the others are right."""
    p = Paged([1, 60, 3], [700, 90, 50], 2, 64, 16, cache, seed=4, extra_table=0)
    p.table[0, 7] = p.n_pages           # seen by the single token
    p.table[1, 4] = -3                  # positions 64 .. 79: the later rows
    Call(p, 4, dt).run().check()
    p.lens[2] = 16 * p.width + 1        # one token past the table
    p.table[2, :] = p.table[0, 0]
    Call(p, 4, dt).run().check()
    p.table[0, :] = -1                  # nothing to read at all
    Call(p, 4, dt).run().check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_scores_of_infinity(dt):
    """A query of infinities, keys that give -infinity everywhere, and large scores that differ little."""
    p = Paged([4], [40], 1, 32, 16, "bf16" if dt == "bf16" else "f32", seed=8)
    a = Call(p, 1, dt, tail=0)
    a.q[1] *= 1e4
    a.run().check()
    for j in range(40):
        row = np.abs(np.random.default_rng(j).standard_normal(32)) + 0.1
        p.set_row("k", 0, j, 0, row)
    a.q[2] = -math.inf   # every score is -infinity: NaN, as its softmax
    a.q[3] = math.nan
    a.run().check()


def test_long_rows_of_values_near_the_largest():
    """Sums of 3000 weights on values of 1e38 do not overflow."""
    p = Paged([1], [3000], 1, 64, 16, "f32", seed=1)
    t = p.pool["v"][0]
    t.copy_(t.sign() * 1e38)
    p.v = t.double().cpu().numpy()
    a = Call(p, 1, "f32", q=torch.zeros((4, 64))).run()
    assert torch.isfinite(a.o[0]).all()
    a.check()


def test_pools_past_four_gigabytes():
    """Page and element offsets past 2^31 and 2^32: pages at both ends of a pool of 6 GB."""
    hd, Hkv, ps = 128, 8, 64
    n_pages = 6 * 2 ** 30 // (ps * Hkv * hd * 2)
    p = Paged([2, 5], [700, 130], Hkv, hd, ps, "bf16", seed=3)
    at = np.linspace(0, n_pages - 1, p.n_pages).astype(np.int64)[::-1].copy()
    for name in "kv":
        small, _ = p.pool[name]
        big = torch.empty((n_pages, Hkv, ps, hd), dtype=torch.bfloat16, device="cuda")
        big[torch.from_numpy(at).cuda()] = small
        p.pool[name] = big, None
    a = Call(p, 8, "bf16")
    plain_table, plain_pages = p.table, p.n_pages
    p.table = np.where(plain_table < plain_pages, at[np.minimum(plain_table, plain_pages - 1)], 2 ** 31 - 7).astype(np.int32)
    p.n_pages = n_pages
    a.run()
    x = torch.randn((a.T, 2 * Hkv * hd), device="cuda").bfloat16()
    call("aic_hip_kv_write", p.struct(), ptr(x), ptr(x) + Hkv * hd * 2, 2 * Hkv * hd, ptr(p.dev_offs), ptr(p.dev_lens), p.B, a.T, CODE["bf16"], stream())
    y = torch.zeros_like(x)
    call("aic_hip_kv_read", p.struct(), ptr(y), ptr(y) + Hkv * hd * 2, 2 * Hkv * hd, ptr(p.dev_offs), ptr(p.dev_lens), p.B, a.T, CODE["bf16"], stream())
    assert torch.equal(x[:7], y[:7]) and (y[7:] == 0).all()
    for b in range(p.B):  # the new rows stand where the table says
        page, slot = p.place(b, p.lens[b] - 1)
        assert torch.equal(p.pool["k"][0][page, :, slot].reshape(-1), x[p.offs[b + 1] - 1, :Hkv * hd])
    p.table, p.n_pages = plain_table, plain_pages
    a.check()


def test_many_sequences():
    """More sequences than a wave has lanes, most of them without rows."""
    rng = np.random.default_rng(5)
    ns = [int(n) for n in rng.integers(0, 4, 200) * (rng.random(200) < 0.5)]
    p = Paged(ns, [n + int(x) for n, x in zip(ns, rng.integers(0, 40, 200))], 1, 32, 8, "bf16", seed=6, first=2)
    Call(p, 2, "bf16").run().check()


def test_captured_and_replayed():
    """Two graphs and eager calls in turn, each graph with its own workspace; the third without one.  New lengths and queries
    in the same buffers reach a replay."""
    ps = [Paged([1, 1], [2100, 900], 2, 64, 16, c, seed=i) for i, c in enumerate(["bf16", "e4m3", "bf16"])]
    calls = [Call(p, 4, "bf16", seed=i) for i, p in enumerate(ps)]
    works = [torch.empty(calls[i].bytes(), dtype=torch.uint8, device="cuda") for i in range(2)] + [None]
    eager = Call(ps[0], 4, "bf16", seed=9)
    s = torch.cuda.Stream()
    structs = [p.struct() for p in ps]

    def launch(a, c, ws, st):
        p = a.p
        call("aic_hip_attn_paged", c, ptr(a.q), a.ld, ptr(a.o), a.ld, ptr(a.lse), ptr(p.dev_offs), ptr(p.dev_lens), *a.sizes(), a.H, 0,
             a.scale, ptr(ws), 0 if ws is None else ws.numel(), CODE["bf16"], st)

    torch.cuda.synchronize()
    graphs = []
    for a, c, ws in zip(calls, structs, works):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            launch(a, c, ws, s.cuda_stream)
        graphs.append(g)
    for turn in range(3):
        for a in calls:
            a.buf.fill_(7.0)
            a.lse.fill_(7.0)
            a.q.copy_(torch.randn(a.q.shape, generator=torch.Generator().manual_seed(turn)))
        for i, a in enumerate(calls):
            a.p.lens = [2100 - 300 * turn - i, 900 + turn]
            a.p.dev_lens.copy_(torch.tensor(a.p.lens))
        torch.cuda.synchronize()
        for g in graphs:
            with torch.cuda.stream(s):
                g.replay()
        launch(eager, structs[0], None, s.cuda_stream)
        torch.cuda.synchronize()
        for a in calls:
            lens = list(a.p.lens)
            a.p.lens = [min(n, a.p.ps * int((a.p.table[b] < a.p.n_pages).sum())) for b, n in enumerate(lens)]
            assert a.p.lens == lens
            a.check()
    _lib.call("aic_hip_mem_release_stream", s.cuda_stream)


def test_streams_do_not_share_results():
    """Two streams of split calls at once, each from the library's scratch of its own stream."""
    ps = [Paged([1] * 3, [1500 + i, 700, 30], 2, 64, 16, "bf16", seed=i) for i in range(2)]
    calls = [Call(p, 8, "bf16", seed=i) for i, p in enumerate(ps)]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(5):
        for a, s in zip(calls, streams):
            a.run(st=s.cuda_stream)
    torch.cuda.synchronize()
    for a in calls:
        a.check()
    for s in streams:
        _lib.call("aic_hip_mem_release_stream", s.cuda_stream)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,L", [(1, 300), (3, 300), (60, 300), (1, 3000)])
def test_e4m3_rows_of_very_different_size(dt, n, L):
    """A few cached rows 2^60 times the others, seen and hidden, and rows of 2^-100: a hidden row costs a visible one
    nothing, and small rows keep their digits."""
    p = Paged([n], [L], 1, 64, 16, "e4m3", seed=n + L)
    for name in "kv":
        codes, exps = p.pool[name]
        for pos, by in ((3, 60), (17, -100), (L - 1, 60), (L - n // 2 - 1, 30), (40, -60)):
            if name == "k" and by > 0:
                by = -by  # large scores would leave one key only
            page, slot = p.place(0, pos)
            exps[page, 0, slot] += by
            getattr(p, name)[page, 0, slot] *= 2.0 ** by
    Call(p, 2, dt).run().check()
    small = Paged([n], [L], 1, 64, 16, "e4m3", seed=n + L)
    codes, exps = small.pool["v"]
    exps -= 110
    small.v *= 2.0 ** -110
    a = Call(small, 2, dt).run()
    a.check()
    assert (a.o[:n, :128] != 0).any()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n,L", [(1, 511), (1, 512), (4, 513), (1, 700), (2, 1023), (1, 1024), (1, 1025), (40, 512), (33, 700), (200, 1300)])
def test_workspaces_are_not_overrun(dt, cache, n, L):
    """Around the lengths where the forms change: nothing behind the bytes asked for is written."""
    p = Paged([n, 1], [L, L // 2], 1, 64, 24, cache, seed=L)
    a = Call(p, 8, dt)
    size = a.bytes()
    ws = torch.full((size + (1 << 20),), 0xa5, dtype=torch.uint8, device="cuda")
    c = p.struct()
    call("aic_hip_attn_paged", c, ptr(a.q), a.ld, ptr(a.o), a.ld, ptr(a.lse), ptr(p.dev_offs), ptr(p.dev_lens), *a.sizes(), a.H, 0, a.scale,
         ptr(ws), size, CODE[dt], stream())
    a.check()
    assert (ws[size:] == 0xa5).all()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n,L,ps", [(1, 1500, 1), (40, 1500, 1), (2, 4000, 3), (70, 4000, 3), (1, 2100, 65536), (40, 700, 65536), (1, 1900, 17)])
def test_page_ids_of_long_caches(dt, cache, n, L, ps):
    """More pages than their ids' place in the kernels holds at a time, and one page larger than the cache."""
    p = Paged([n], [L], 1, 32, ps, cache, seed=ps)
    Call(p, 2, dt).run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens,window", [([300, 17], [1500, 900], 0), ([300, 17], [1500, 900], 400), ([130], [1000], 65), ([257], [257], 0)])
@pytest.mark.parametrize("H,Hkv,hd,ps", [(4, 2, 128, 16), (3, 3, 64, 24)])
def test_chunks_of_long_prompts(dt, cache, ns, lens, window, H, Hkv, hd, ps):
    """Several query tiles and many tiles of keys that every row sees whole, between masked ones."""
    p = Paged(ns, lens, Hkv, hd, ps, cache, seed=hd + window)
    Call(p, H, dt, window).run().check()


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "e4m3")])
def test_many_rows_and_heads_fill_the_card(dt, cache):
    """Enough blocks that nothing is split: 700 rows of 32 heads."""
    p = Paged([600, 100], [600, 150], 16, 32, 16, cache, seed=1)
    a = Call(p, 32, dt, with_lse=False).run()
    q = a.q[:, :a.w].double().cpu().numpy().reshape(a.T, 32, 32)
    some = Paged.__new__(Paged)  # every eighth head against the definition
    some.__dict__.update(p.__dict__)
    for h in range(0, 32, 8):
        some.k, some.v, some.Hkv = p.k[:, h // 2:h // 2 + 1], p.v[:, h // 2:h // 2 + 1], 1
        got = host(a.o.contiguous()).reshape(a.T, 32, 32)[:, h:h + 1]
        check_attention(got, None, some, q[:, h:h + 1], 1, 0, a.scale, dt)


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 62])
@pytest.mark.parametrize("n,L", [(3, 1), (40, 20), (300, 220), (5, 0)])
def test_windows_up_to_the_largest(dt, cache, window, n, L):
    """More rows than cached tokens: the first ones stand before position 0."""
    p = Paged([n, 2], [L, 50], 1, 32, 16, cache, seed=n)
    Call(p, 1, dt, window).run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n", [1, 40])
def test_the_longest_cache(dt, cache, n):
    """2^31 - 4096 positions: a page, the same page over and over, and a last one cut short.  The keys of the middle lie
    40 below the others in the scores: together they weigh less than 2^31 e^-35 = 1.4e-6 of the others, whose
    scores differ by less than 5, and as much is added to the tolerance."""
    ps, L = 65536, 2 ** 31 - 4096
    p = Paged([n], [3 * ps], 1, 32, ps, cache, seed=n)
    (first, mid, last), p.width, p.lens = p.table[0, :3].tolist(), 2 ** 15, [L]
    p.table = np.full((1, p.width), mid, np.int32)
    p.table[0, 0], p.table[0, -1] = first, last
    k = p.k * 0.125
    k[..., 0] = 0.0
    k[mid, ..., 0] = -40.0
    if cache == "e4m3":
        codes, exps = e4m3_encode(k)
        p.pool["k"], p.k = (torch.from_numpy(codes).cuda(), torch.from_numpy(exps).cuda()), e4m3_decode(codes, exps)
    else:
        t = torch.from_numpy(k).to(TORCH[cache])
        p.pool["k"], p.k = (t.cuda(), None), t.double().numpy()
    q = torch.from_numpy(np.random.default_rng(n).standard_normal((n + 3, 32)).clip(-2, 2))
    q[:, 0] = 32.0 ** 0.5
    a = Call(p, 1, dt, q=q).run()
    torch.cuda.synchronize()
    short = Paged.__new__(Paged)  # without the middle
    short.__dict__.update(p.__dict__)
    short.table, short.width, short.lens = np.array([[first, last]], np.int32), 2, [2 * ps - 4096]
    q = a.q.double().cpu().numpy().reshape(a.T, 1, 32)
    o, lse, ab, sb = attention(short, q, 1, 0, a.scale)
    got, got_lse = host(a.o).reshape(a.T, 1, 32).astype(np.float64), host(a.lse).astype(np.float64)
    mass = 2.0 ** 31 * math.exp(-35)
    tol = (4 * sb[:n, :, None] + 2.0 ** -18) * ab[:n] + (HALF[dt] * np.abs(o[:n]) + (HALF["bf16"] * ab[:n] if dt == "bf16" else 0)) * 1.01
    assert (np.abs(got - o)[:n] <= tol + 2 * mass * np.abs(p.v).max()).all()
    assert (np.abs(got_lse - lse)[:n] <= 2 * sb[:n] + 2.0 ** -17 + 2.0 ** -22 * np.abs(lse[:n]) + mass).all()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("B,Hkv", [(64, 1), (70, 1), (128, 1), (129, 1), (257, 2), (700, 1)])
def test_large_batches_with_a_few_long_caches(dt, cache, B, Hkv):
    """One to three rows of each sequence, some without rows or without a cache, a few of them long enough to be divided."""
    rng = np.random.default_rng(B)
    ns = rng.integers(0, 4, B)
    lens = np.where(rng.random(B) < 0.1, 0, ns + rng.integers(0, 90, B))
    for b, n in ((0, 2300), (B // 2, 4100), (B - 1, 3000)):
        ns[b], lens[b] = 2, n
    p = Paged(ns.tolist(), lens.tolist(), Hkv, 32, 16, cache, seed=B)
    a = Call(p, 2, dt).run()
    a.check()
    first = a.o.clone(), a.lse.clone()
    a.run()
    torch.cuda.synchronize()
    assert torch.equal(first[0], a.o) and torch.equal(first[1], a.lse)


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens", [([1, 2], [700, 1300]), ([40, 150], [700, 300])])
def test_pools_past_four_gigabytes_in_every_form(dt, cache, ns, lens):
    """The first pages at the far end of pools of 6 GB."""
    hd, Hkv, ps = 64, 4, 64
    p = Paged(ns, lens, Hkv, hd, ps, cache, seed=sum(ns))
    small, n_pages = p.n_pages, 6 * 2 ** 30 // (ps * Hkv * hd * TORCH[cache].itemsize)
    at = np.linspace(n_pages - 1, 0, small).astype(np.int64)
    for name in "kv":
        pair = []
        for t in p.pool[name]:
            big = None
            if t is not None:
                big = torch.empty((n_pages, *t.shape[1:]), dtype=t.dtype, device="cuda")
                big[torch.from_numpy(at).cuda()] = t
            pair.append(big)
        p.pool[name] = tuple(pair)
    table = p.table
    p.table = np.where(table < small, at[np.minimum(table, small - 1)], 2 ** 31 - 7).astype(np.int32)
    p.n_pages = n_pages
    a = Call(p, 4, dt).run()
    torch.cuda.synchronize()
    p.table, p.n_pages = table, small
    a.check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("max_q,max_len", [(1, 1), (1, 5000), (7, 64)])
def test_larger_than_promised_in_every_form(dt, cache, max_q, max_len):
    p = Paged([20, 1, 90, 0, 9], [900, 2300, 95, 40, 700], 2, 32, 16, cache, seed=max_q)
    a = Call(p, 4, dt)
    a.sizes = lambda: (p.B, a.T, max_q, max_len)
    a.run().check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n", [1, 3, 40, 200])
@pytest.mark.parametrize("own", [True, False])
def test_replays_of_every_form(dt, cache, n, own):
    """With a workspace and without: three replays between eager calls on other queries and lengths, equal to the eager
    result on the same."""
    p = Paged([n, 1], [1700, 900], 2, 64, 16, cache, seed=n)
    a = Call(p, 2, dt)
    ws = torch.empty(max(a.bytes(), 16), dtype=torch.uint8, device="cuda") if own else None
    c = p.struct()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def launch():
        call("aic_hip_attn_paged", c, ptr(a.q), a.ld, ptr(a.o), a.ld, ptr(a.lse), ptr(p.dev_offs), ptr(p.dev_lens), *a.sizes(), a.H, 0, a.scale,
             ptr(ws), 0 if ws is None else ws.numel(), CODE[dt], s.cuda_stream)

    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        launch()
    sizes = a.sizes()
    a.sizes = lambda: sizes
    for turn in range(3):
        a.q.copy_(torch.randn(a.q.shape, generator=torch.Generator().manual_seed(turn)))
        p.lens = [1700 - 200 * turn, 900 - turn]
        p.dev_lens.copy_(torch.tensor(p.lens))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        a.check()
        a.buf.fill_(7.0)
        a.lse.fill_(7.0)
        launch()
        torch.cuda.synchronize()
        a.check()
    _lib.call("aic_hip_mem_release_stream", s.cuda_stream)


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens,H,Hkv,window", [([8, 5, 1], [2600, 1500, 40], 8, 1, 0), ([33, 64], [1400, 70], 1, 1, 0), ([64, 2], [500, 300], 2, 2, 90),
                                                  ([65], [1300], 1, 1, 0)])
def test_two_groups_of_rows(dt, cache, ns, lens, H, Hkv, window):
    """33 to 65 rows per key/value head of 128."""
    p = Paged(ns, lens, Hkv, 128, 16, cache, seed=len(ns))
    Call(p, H, dt, window).run().check()
