"""Writing into and reading from the paged key/value cache (csrc/kernels/paged_kv.hip), byte for byte against the
definition: shuffled pages, odd page sizes, empty sequences and positions without a place."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from tests.gpu_util import call, ptr, stream  # noqa: E402
from tests.paged_ref import CODE, TORCH, Paged, e4m3_decode, e4m3_encode  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


# (ns, lens, Hkv, hd, page size, columns of the rows beyond the heads, elements before the rows)
BATCHES = [([1], [1], 1, 32, 1, 0, 0), ([1, 1, 1], [5, 16, 17], 3, 64, 16, 8, 0), ([7, 0, 300, 1], [9, 4, 300, 64], 2, 128, 24, 0, 0),
           ([40, 3], [33, 2], 4, 128, 7, 3, 1), ([0, 0, 5, 0], [0, 3, 5, 0], 1, 64, 128, 0, 4), ([33] * 9, [40] * 9, 2, 32, 64, 8, 0)]
TYPES = [("f32", "f32"), ("f32", "e4m3"), ("bf16", "bf16"), ("bf16", "e4m3")]


def _rows(p, dt, pad, shift, seed, tail=5):
    """k and v as columns of one matrix, with `tail` rows behind the last sequence."""
    T, w = p.offs[-1] + tail, p.Hkv * p.hd
    ld = 2 * w + pad
    buf = torch.empty(T * ld + shift + 16, dtype=TORCH[dt], device="cuda")
    x = buf[shift:shift + T * ld].view(T, ld)
    g = torch.Generator(device="cuda").manual_seed(seed)
    x.copy_(torch.randn((T, ld), generator=g, device="cuda").to(TORCH[dt]))
    return buf, x, ld, T


def _filled(p):
    """Every byte of the pools to a mark, to see what is written."""
    for name in "kv":
        for t in p.pool[name]:
            if t is not None:
                t.view(torch.uint8).fill_(0x5a)


def _expect(p, x, dt):
    w, want = p.Hkv * p.hd, {}
    host = x.double().cpu().numpy()
    for i, name in enumerate("kv"):
        pool, exps = (None if t is None else t.cpu() for t in p.pool[name])
        for b in range(p.B):
            for r in range(p.ns[b]):
                at = p.place(b, p.lens[b] - p.ns[b] + r)
                if at is None:
                    continue
                row = host[p.offs[b] + r, i * w:(i + 1) * w].reshape(p.Hkv, p.hd)
                if p.cache == "e4m3":
                    codes, e = e4m3_encode(row)
                    pool[at[0], :, at[1]] = torch.from_numpy(codes)
                    exps[at[0], :, at[1]] = torch.from_numpy(e)
                else:
                    pool[at[0], :, at[1]] = torch.from_numpy(row).to(TORCH[dt])
        want[name] = pool, exps
    return want


def _write(p, x, ld, T, dt):
    w, size = p.Hkv * p.hd, x.element_size()
    call("aic_hip_kv_write", p.struct(), ptr(x), ptr(x) + w * size, ld, ptr(p.dev_offs), ptr(p.dev_lens), p.B, T, CODE[dt], stream())


def _same(p, want):
    for name in "kv":
        for got, exp in zip(p.pool[name], want[name]):
            if got is not None:
                assert torch.equal(got.cpu().view(torch.uint8), exp.view(torch.uint8)), name


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens,Hkv,hd,ps,pad,shift", BATCHES)
def test_write_and_read_back(dt, cache, ns, lens, Hkv, hd, ps, pad, shift):
    p = Paged(ns, lens, Hkv, hd, ps, cache, seed=hd + ps)
    _, x, ld, T = _rows(p, dt, pad, shift, seed=len(ns))
    _filled(p)
    want = _expect(p, x, dt)
    _write(p, x, ld, T, dt)
    _same(p, want)

    buf, y, _, _ = _rows(p, dt, pad, shift, seed=99)
    before = buf.clone()
    w, size = Hkv * hd, y.element_size()
    call("aic_hip_kv_read", p.struct(), ptr(y), ptr(y) + w * size, ld, ptr(p.dev_offs), ptr(p.dev_lens), p.B, T, CODE[dt], stream())
    ref = before.clone()
    rows = ref[shift:shift + T * ld].view(T, ld)
    for b in range(p.B):
        for r in range(ns[b]):
            at = p.place(b, lens[b] - ns[b] + r)
            for i, name in enumerate("kv"):
                pool, exps = p.pool[name]
                if at is None:
                    val = np.zeros((Hkv, hd))
                elif cache == "e4m3":
                    val = e4m3_decode(pool[at[0], :, at[1]].cpu().numpy(), exps[at[0], :, at[1]].cpu().numpy())
                else:
                    val = pool[at[0], :, at[1]].double().cpu().numpy()
                rows[p.offs[b] + r, i * w:(i + 1) * w] = torch.from_numpy(val.reshape(-1)).to(TORCH[dt]).cuda()
    assert torch.equal(buf.view(torch.uint8), ref.view(torch.uint8))  # rows behind the last sequence and the padding too


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_e4m3_of_extreme_rows(dt):
    """Zeros, the largest and smallest numbers, ties between codes, rows whose amax is just at, above and below
    448 times a power of two, infinities and NaN."""
    hd = 64
    rows = np.zeros((12, hd), np.float64)
    rows[1, 3] = 3.3e38
    rows[2] = 2.0 ** -133 * (np.arange(hd) - 20)            # subnormal
    rows[3, :3] = [1.75, 1.0, -1.75]                        # amax = 448 * 2^-8 exactly
    rows[4, :3] = [1.7578125, 1.0, -1.75]                   # one bf16 step above
    rows[5, :3] = [1.7421875, 1.0, -1.75 + 2 ** -7]
    rows[6] = 256.0 * (1 + (np.arange(hd) % 16) / 16.0)     # odd sixteenths lie between two codes
    rows[7] = rows[6] / 1024 - 0.3
    rows[8, :5] = [np.inf, -np.inf, np.nan, 5.0, -0.0]
    rows[9] = np.nan
    rows[10] = 2.0 ** (np.arange(hd) % 30 - 20) * np.where(np.arange(hd) % 3, 1, -1)  # down to codes' subnormals
    rows[11, 0] = 2.0 ** -126
    p = Paged([12], [12], 1, hd, 5, "e4m3", seed=1)
    x = torch.from_numpy(np.concatenate([rows, -rows], 1)).to(TORCH[dt]).cuda()
    _filled(p)
    want = _expect(p, x, dt)
    _write(p, x, 2 * hd, 12, dt)
    for name in "kv":
        got, e = (t.cpu() for t in p.pool[name])
        codes, we = want[name]
        nan = (codes & 127) == 127
        assert torch.equal((got & 127) == 127, nan)
        assert torch.equal(got[~nan], codes[~nan]) and torch.equal(e, we)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_places_without_a_page(cache):
    """Ids outside the pool and positions past the page table's row: not written, read as zeros."""
    p = Paged([6, 8], [40, 8], 2, 64, 4, cache, seed=3, extra_table=0)
    p.table[0, 9] = -1                     # positions 36 .. 39 of sequence 0
    p.table[1, 0] = p.n_pages              # positions 0 .. 3 of sequence 1
    p.lens[1] = 8 + 4 * (p.width - 1)      # its rows reach past the table's width
    p.ns[1] = 8
    for j in range(2, p.width):
        p.table[1, j] = p.table[0, j % 9]  # valid ids elsewhere
    p.table[1, p.width - 1] = p.table[0, 1]
    _, x, ld, T = _rows(p, "bf16", 0, 0, seed=4)
    _filled(p)
    want = _expect(p, x, "bf16")
    _write(p, x, ld, T, "bf16")
    _same(p, want)
    y = torch.ones_like(x)
    w = p.Hkv * p.hd
    call("aic_hip_kv_read", p.struct(), ptr(y), ptr(y) + 2 * w, ld, ptr(p.dev_offs), ptr(p.dev_lens), p.B, T, CODE["bf16"], stream())
    for b in range(p.B):
        for r in range(p.ns[b]):
            if p.place(b, p.lens[b] - p.ns[b] + r) is None:
                assert (y[p.offs[b] + r] == 0).all()
            else:
                assert (y[p.offs[b] + r] != 0).any()
    assert (y[p.offs[-1]:] == 1).all()


def test_many_sequences_and_rows_before_the_first():
    """More sequences than a block has threads, most without rows, behind three rows of nobody."""
    rng = np.random.default_rng(5)
    ns = [int(n) for n in rng.integers(0, 3, 700) * (rng.random(700) < 0.4)]
    p = Paged(ns, [n + 3 for n in ns], 1, 32, 4, "bf16", seed=6, first=3)
    _, x, ld, T = _rows(p, "bf16", 0, 0, seed=7)
    _filled(p)
    want = _expect(p, x, "bf16")
    _write(p, x, ld, T, "bf16")
    _same(p, want)
