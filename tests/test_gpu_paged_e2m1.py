"""The paged cache in 4 bits (csrc/kernels/paged_kv.hip, attention_paged*.hip): writing and reading byte for byte
against the definition, and attention over it against 64 bits at the sizes, masks and values where its tiles can go wrong."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests.gpu_util import call, ptr, stream  # noqa: E402
from tests.paged_codes_ref import Cache, e2m1_decode, e2m1_encode  # noqa: E402
from tests.paged_ref import CODE, TORCH  # noqa: E402
from tests.test_gpu_attn_paged import CASES, Call  # noqa: E402
from tests.test_gpu_paged_kv import BATCHES, _filled, _rows  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def _written(p, x):
    """The pools after writing the rows x (k, then v, side by side)."""
    w, want = p.Hkv * p.hd, {}
    host = x.double().cpu().numpy()
    for i, name in enumerate("kv"):
        pool, exps = (t.cpu().numpy() for t in p.pool[name])
        for b in range(p.B):
            for r in range(p.ns[b]):
                at = p.place(b, p.lens[b] - p.ns[b] + r)
                if at is not None:
                    row = host[p.offs[b] + r, i * w:(i + 1) * w].reshape(p.Hkv, p.hd)
                    pool[at[0], :, at[1]], exps[at[0], :, at[1]] = e2m1_encode(row)
        want[name] = pool, exps
    return want


def _same(p, want):
    for name in "kv":
        for got, exp in zip(p.pool[name], want[name]):
            assert np.array_equal(got.cpu().numpy(), exp), name


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("ns,lens,Hkv,hd,ps,pad,shift", BATCHES)
def test_write_and_read_back(dt, ns, lens, Hkv, hd, ps, pad, shift):
    p = Cache(ns, lens, Hkv, hd, ps, "e2m1", seed=hd + ps)
    _, x, ld, T = _rows(p, dt, pad, shift, seed=len(ns))
    _filled(p)
    want = _written(p, x)
    w, size = Hkv * hd, x.element_size()
    call("aic_hip_kv_write", p.struct(), ptr(x), ptr(x) + w * size, ld, ptr(p.dev_offs), ptr(p.dev_lens), p.B, T, CODE[dt], stream())
    _same(p, want)

    buf, y, _, _ = _rows(p, dt, pad, shift, seed=99)
    ref = buf.clone()
    call("aic_hip_kv_read", p.struct(), ptr(y), ptr(y) + w * size, ld, ptr(p.dev_offs), ptr(p.dev_lens), p.B, T, CODE[dt], stream())
    rows = ref[shift:shift + T * ld].view(T, ld)
    for b in range(p.B):
        for r in range(ns[b]):
            at = p.place(b, lens[b] - ns[b] + r)
            for i, name in enumerate("kv"):
                val = np.zeros((Hkv, hd)) if at is None else e2m1_decode(*(t[at[0], :, at[1]] for t in want[name]))
                rows[p.offs[b] + r, i * w:(i + 1) * w] = torch.from_numpy(val.reshape(-1)).to(TORCH[dt]).cuda()
    assert torch.equal(buf.view(torch.uint8), ref.view(torch.uint8))  # rows behind the last sequence and the padding too


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_extreme_rows(dt):
    """Zeros of both signs, the largest and smallest numbers, ties between codes, groups whose amax is just at, above and below 6 times
    a power of two, infinities and NaN; their neighbours' groups as if alone."""
    hd = 64
    rows = np.zeros((13, hd), np.float64)
    rows[0, 1] = -0.0
    rows[1, 3] = 3.3e38                                     # past 6 * 2^125
    rows[1, 4:8] = [2.55e38, 1e38, -3e37, 1e37]
    rows[2] = 2.0 ** -133 * (np.arange(hd) - 20)            # subnormal
    rows[3, :3] = [1.5, 1.0, -1.5]                          # amax = 6 * 2^-2 exactly
    rows[4, :3] = [1.5078125, 1.0, -1.5]                    # one bf16 step above
    rows[5, :3] = [1.4921875, 1.0, -1.4921875]
    rows[6] = np.arange(hd) % 32 * 0.25                     # up to 7.75: power 1, ties at odd quarters and between 4 and 6
    rows[7] = np.where(np.arange(hd) % 2, -1, 1) * (np.arange(hd) % 25) * 0.25  # up to 6: power 0, every tie
    rows[8, :5] = [np.inf, -np.inf, np.nan, 5.0, -0.0]      # the second half's group is fine
    rows[8, 40:] = np.arange(24)
    rows[9] = np.nan
    rows[10] = 2.0 ** (np.arange(hd) % 30 - 20) * np.where(np.arange(hd) % 3, 1, -1)
    rows[11, 0] = 2.0 ** -126
    rows[12, 33] = -2.0 ** -133
    p = Cache([13], [13], 1, hd, 5, "e2m1", seed=1)
    x = torch.from_numpy(np.concatenate([rows, -rows], 1)).to(TORCH[dt]).cuda()
    _filled(p)
    want = _written(p, x)
    call("aic_hip_kv_write", p.struct(), ptr(x), ptr(x) + hd * x.element_size(), 2 * hd, ptr(p.dev_offs), ptr(p.dev_lens), 1, 13, CODE[dt],
         stream())
    _same(p, want)
    y = torch.empty_like(x)
    call("aic_hip_kv_read", p.struct(), ptr(y), ptr(y) + hd * x.element_size(), 2 * hd, ptr(p.dev_offs), ptr(p.dev_lens), 1, 13, CODE[dt],
         stream())
    for i, name in enumerate("kv"):
        val = np.stack([e2m1_decode(*(t[p.place(0, j)[0], 0, p.place(0, j)[1]] for t in want[name])) for j in range(13)])
        got = y[:, i * hd:(i + 1) * hd].double().cpu().numpy()
        assert np.array_equal(got, val, equal_nan=True)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_every_code_and_power(dt):
    """Reading: all 16 codes with powers from the least to the largest."""
    p = Cache([252], [252], 1, 32, 16, "e2m1", seed=2)
    codes, exps = (t.cpu().numpy() for t in p.pool["k"])
    for j in range(252):
        page, slot = p.place(0, j)
        codes[page, 0, slot] = np.arange(16, dtype=np.uint8) * 16 + (np.arange(16, dtype=np.uint8) + j) % 16
        exps[page, 0, slot] = j + 1
    p.set_codes("k", codes, exps)
    y = torch.empty((2, 252, 32), dtype=TORCH[dt], device="cuda")
    call("aic_hip_kv_read", p.struct(), ptr(y), ptr(y[1]), 32, ptr(p.dev_offs), ptr(p.dev_lens), 1, 252, CODE[dt], stream())
    assert np.array_equal(y[0].double().cpu().numpy(), p.rows("k", 0, 0))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("ns,lens,H,Hkv,hd,ps,window,pad,shift", CASES)
def test_attention(dt, ns, lens, H, Hkv, hd, ps, window, pad, shift):
    p = Cache(ns, lens, Hkv, hd, ps, "e2m1", seed=hd + len(ns))
    Call(p, H, dt, window, pad, shift).run().check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("ns,lens,H,Hkv,hd", [([1, 1, 1], [4100, 700, 1], 8, 2, 64), ([3, 8, 0], [2500, 1100, 900], 4, 4, 32),
                                              ([60, 1], [1500, 3000], 2, 1, 128), ([1] * 70, [2100] * 69 + [5000], 2, 1, 128),
                                              ([16, 3], [900, 1400], 4, 1, 128), ([300, 7], [1300, 1024], 4, 2, 128)])
def test_keys_split_among_blocks(dt, ns, lens, H, Hkv, hd):
    """Few rows over long caches: the split form with the call's own workspace and with the stream's, exactly alike, with and
    without lse."""
    p = Cache(ns, lens, Hkv, hd, 16, "e2m1", seed=hd)
    a = Call(p, H, dt)
    assert a.bytes() > 0
    ws = torch.full((a.bytes(),), 0xff, dtype=torch.uint8, device="cuda")  # NaN in every place
    a.run(ws).check()
    b = Call(p, H, dt, with_lse=False).run().check()
    assert torch.equal(a.o, b.o)
    with pytest.raises(_lib.AicError, match="workspace"):
        Call(p, H, dt).run(ws[:a.bytes() - 16])


@pytest.mark.parametrize("ns,lens,H,Hkv,hd,ps,window", [
    ([10] * 27, [3900] * 14 + [2700] * 13, 8, 2, 64, 24, 0), ([33, 0] + [40] * 18, [11200] + [9] + [4000] * 18, 1, 1, 128, 16, 700),
    ([5] * 100, [2003] * 100, 16, 2, 32, 16, 0), ([1] * 200, [4090, 1] * 100, 2, 1, 128, 32, 0)])
def test_batches_with_many_keys(ns, lens, H, Hkv, hd, ps, window):
    """Two groups of rows over one cache, divided and whole."""
    Call(Cache(ns, lens, Hkv, hd, ps, "e2m1", seed=hd), H, "bf16", window).run().check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,L,H,Hkv,hd,ps", [(1, 300, 8, 1, 128, 16), (1, 2000, 1, 1, 64, 24), (40, 100, 2, 1, 64, 16), (150, 400, 2, 1, 128, 64),
                                             (3, 700, 2, 1, 32, 8)])
def test_groups_of_nan(dt, n, L, H, Hkv, hd, ps):
    """NaN groups of a key and of a value: the rows that see them show them, in all columns or in the group's; others do not."""
    for name, pos in (("k", L - n // 2 - 1), ("v", L - 1), ("v", L - n - 1), ("k", 0), ("v", 17)):
        p = Cache([n], [L], Hkv, hd, ps, "e2m1", seed=L)
        codes, exps = (t.cpu().numpy() for t in p.pool[name])
        page, slot = p.place(0, pos)
        exps[page, 0, slot, hd // 32 - 1] = 255
        p.set_codes(name, codes, exps)
        Call(p, H, dt).run().check()


def test_stale_values_behind_a_sequence():
    """Slots past a sequence's length in its last page, and all pages of nobody, hold NaN."""
    p = Cache([1, 30, 2, 200], [5, 37, 600, 300], 2, 64, 64, "e2m1", seed=2)
    used = np.zeros((p.n_pages, p.ps), bool)
    for b in range(p.B):
        for j in range(p.lens[b]):
            used[p.place(b, j)] = True
    free = torch.from_numpy(~used).cuda()
    for name in "kv":
        for t in p.pool[name]:
            t.permute(0, 2, 1, 3)[free] = 0xff
    Call(p, 4, "bf16").run().check()
    Call(p, 4, "f32").run().check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_pages_outside_the_pool(dt, hd):
    """Rows that see a position whose page id is out of range, or past the table's row, are NaN; the others are right."""
    p = Cache([1, 60, 3], [700, 90, 50], 2, hd, 16, "e2m1", seed=4, extra_table=0)
    p.table[0, 7] = p.n_pages           # seen by the single token
    p.table[1, 4] = -3                  # positions 64 .. 79: the later rows
    Call(p, 4, dt).run().check()
    p.ns[1] = p.lens[1] = 0             # few rows in every sequence
    p.offs = [0, 1, 1, 4]
    Call(p, 4, dt).run().check()
    p.lens[2] = 16 * p.width + 1        # one token past the table
    p.table[2, :] = p.table[0, 0]
    Call(p, 4, dt).run().check()
    p.table[0, :] = -1                  # nothing to read at all
    Call(p, 4, dt).run().check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,L,H,Hkv,hd", [(1, 3000, 4, 1, 64), (1, 200, 1, 1, 128), (50, 300, 2, 1, 32), (200, 260, 2, 2, 128)])
def test_values_of_all_sizes(dt, n, L, H, Hkv, hd):
    """Values near the largest that the codes hold beside ones of 1e-30: sums do not overflow, small ones keep their digits where the
    large ones' columns are others."""
    p = Cache([n], [L], Hkv, hd, 16, "e2m1", seed=5)
    codes, exps = (t.cpu().numpy() for t in p.pool["v"])
    exps[..., 0] = 252 if hd == 32 else 27
    if hd > 32:
        exps[..., 1] = 252
    p.set_codes("v", codes, exps)
    Call(p, H, dt).run().check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,L,H,Hkv,hd", [(1, 5000, 16, 2, 128), (1, 600, 12, 12, 64), (40, 900, 4, 1, 64), (300, 500, 2, 1, 128)])
def test_captured_and_replayed(dt, n, L, H, Hkv, hd):
    """A graph with a workspace of its own and one without: every replay as the eager call, with eager work between."""
    p = Cache([n, 1], [L, L // 2], Hkv, hd, 16, "e2m1", seed=6)
    for own in (True, False):
        a = Call(p, H, dt)
        ws = torch.zeros(max(a.bytes(), 16), dtype=torch.uint8, device="cuda") if own else None
        a.run(ws).check()
        want = a.o.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        c = p.struct()
        held = p.dev_table, p.dev_offs, p.dev_lens  # the graph's, while later calls make their own
        args = (c, ptr(a.q), a.ld, ptr(a.o), a.ld, ptr(a.lse), ptr(p.dev_offs), ptr(p.dev_lens), *a.sizes(), a.H, a.window, a.scale,
                *((ptr(ws), ws.numel()) if own else (None, 0)), CODE[dt])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call("aic_hip_attn_paged", *args, torch.cuda.current_stream().cuda_stream)
        for _ in range(3):
            a.o[:p.offs[-1], :a.w].zero_()
            graph.replay()
            torch.cuda.synchronize()
            if own:
                assert torch.equal(a.o, want)
            a.check()
            Call(p, H, dt).run()
        del held


@pytest.mark.parametrize("n,L", [(1, 700), (40, 60)])
def test_pools_past_four_gigabytes(n, L):
    """Page, code and exponent offsets past 2^32: pages at both ends of a pool of 5 GB."""
    hd, Hkv, ps = 128, 8, 64
    n_pages = 5 * 2 ** 30 // (ps * Hkv * hd // 2)
    p = Cache([n, 5], [L, 130], Hkv, hd, ps, "e2m1", seed=3)
    at = np.linspace(0, n_pages - 1, p.n_pages).astype(np.int64)[::-1].copy()
    small = {name: tuple(t.clone() for t in p.pool[name]) for name in "kv"}
    dev = torch.from_numpy(at).cuda()
    for name in "kv":
        big = (torch.empty((n_pages, Hkv, ps, hd // 2), dtype=torch.uint8, device="cuda"),
               torch.empty((n_pages, Hkv, ps, hd // 32), dtype=torch.uint8, device="cuda"))
        for t, s in zip(big, small[name]):
            t[dev] = s
        p.pool[name] = big
    values = {name: getattr(p, name) for name in "kv"}

    class Far:
        def __init__(self, x):
            self.x, self.of = x, {int(page): i for i, page in enumerate(at)}

        def __getitem__(self, i):
            return self.x[(self.of[int(i[0])],) + i[1:]]

    p.table = np.where((p.table >= 0) & (p.table < p.n_pages), at[np.clip(p.table, 0, p.n_pages - 1)], p.table).astype(np.int32)
    p.n_pages = n_pages
    for name in "kv":
        setattr(p, name, Far(values[name]))
    for dt in ("bf16", "f32"):
        Call(p, 16, dt).run().check()
