"""Rotating and appending to the paged cache in one call (aic_hip_kv_append, csrc/kernels/paged_kv.hip), bit for bit against the
four operations in fp32 and one rounding."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests.gpu_util import call, ptr, stream  # noqa: E402
from tests.paged_codes_ref import Cache, encode, turn  # noqa: E402
from tests.paged_ref import CODE, TORCH  # noqa: E402
from tests.test_gpu_paged_kv import _filled  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def _tables(n_pos, hd, shift=0):
    c, s = np.empty((n_pos, hd // 2), np.float32), np.empty((n_pos, hd // 2), np.float32)
    call("aic_hip_rope_tables", c.ctypes.data, s.ctypes.data, n_pos, hd, 10000.0)
    dev = []
    for x in (c, s):
        buf = torch.empty(x.size + shift, device="cuda")
        buf[shift:] = torch.from_numpy(x).cuda().view(-1)
        dev.append(buf[shift:])
    return c, s, dev[0], dev[1]


class Append:
    """Fused q, k, v rows with padding, and everything that one call leaves."""

    def __init__(self, p, H, dt, n_pos=None, pad=0, shift=0, tail=4, seed=0, in_place=False, x=None):
        self.p, self.H, self.dt, self.in_place = p, H, dt, in_place
        self.wq, self.wk = H * p.hd, p.Hkv * p.hd
        self.T, self.ld = p.offs[-1] + tail, self.wq + 2 * self.wk + pad
        g = torch.Generator(device="cuda").manual_seed(seed + 3)
        buf = torch.empty(self.T * self.ld + shift + 16, dtype=TORCH[dt], device="cuda")
        self.x = buf[shift:shift + self.T * self.ld].view(self.T, self.ld)
        self.x.copy_(torch.randn((self.T, self.ld), generator=g, device="cuda") if x is None else x)
        self.n_pos = max(p.lens) + 1 if n_pos is None else n_pos
        self.c, self.s, self.dev_c, self.dev_s = _tables(self.n_pos, p.hd, shift)
        self.ldo = self.ld if in_place else self.wq + 8 + pad
        self.out = self.x if in_place else torch.full((self.T, self.ldo), 7.0, dtype=TORCH[dt], device="cuda")
        _filled(p)

    def args(self):
        p, size = self.p, self.x.element_size()
        return (p.struct(), ptr(self.x), self.ld, ptr(self.out), self.ldo, self.H, ptr(self.x) + self.wq * size,
                ptr(self.x) + (self.wq + self.wk) * size, self.ld, ptr(self.dev_c), ptr(self.dev_s), self.n_pos, ptr(p.dev_offs),
                ptr(p.dev_lens), p.B, self.T, CODE[self.dt])

    def expect(self):
        p = self.p
        host, out = self.x.float().cpu().numpy(), self.out.float().cpu().numpy().copy()
        pools = {n: tuple(None if t is None else t.cpu().clone() for t in p.pool[n]) for n in "kv"}
        for b in range(p.B):
            for r in range(p.ns[b]):
                t, pos = p.offs[b] + r, p.lens[b] - p.ns[b] + r
                if pos < 0:
                    continue
                row = host[t, :self.wq + 2 * self.wk].reshape(1, -1, p.hd)
                if pos >= self.n_pos:
                    out[t, :self.wq] = np.nan
                    continue
                heads = self.H + p.Hkv
                turned = turn(row[:, :heads], self.c[pos][None], self.s[pos][None])[0]
                out[t, :self.wq] = turned[:self.H].reshape(-1)
                at = p.place(b, pos)
                if at is None:
                    continue
                for name, y in (("k", turned[self.H:]), ("v", row[0, heads:])):
                    pool, exps = pools[name]
                    if exps is None:
                        pool[at[0], :, at[1]] = torch.from_numpy(y).to(pool.dtype)
                    else:
                        codes, e = encode(y.astype(np.float64), p.cache)
                        pool[at[0], :, at[1]], exps[at[0], :, at[1]] = torch.from_numpy(codes), torch.from_numpy(e)
        return torch.from_numpy(out).to(TORCH[self.dt]), pools

    def check(self):
        before = self.x.clone()
        out, pools = self.expect()
        call("aic_hip_kv_append", *self.args(), stream())
        got = self.out.cpu()
        nan = torch.isnan(out)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[~nan], out[~nan])
        if not self.in_place:
            assert torch.equal(self.x.view(torch.uint8), before.view(torch.uint8))
        for name in "kv":
            for g, e in zip(self.p.pool[name], pools[name]):
                assert g is None or torch.equal(g.cpu().view(torch.uint8), e.view(torch.uint8)), name


TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f32", "e4m3"), ("bf16", "e4m3"), ("f32", "e2m1"), ("bf16", "e2m1")]
# (ns, lens, H, Hkv, hd, page size, columns beyond the heads, elements before the rows)
BATCHES = [([1], [1], 1, 1, 32, 1, 0, 0), ([1, 1, 1], [5, 16, 17], 6, 3, 64, 16, 8, 0), ([7, 0, 300, 1], [9, 4, 300, 64], 2, 2, 128, 24, 0, 0),
           ([40, 3], [33, 2], 4, 4, 128, 7, 3, 1), ([0, 0, 5, 0], [0, 3, 5, 0], 3, 1, 64, 128, 0, 4), ([33] * 9, [400] * 9, 4, 2, 32, 64, 8, 0),
           ([900, 1, 2000], [901, 700, 2100], 16, 8, 128, 64, 0, 0)]


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("ns,lens,H,Hkv,hd,ps,pad,shift", BATCHES)
def test_append(dt, cache, ns, lens, H, Hkv, hd, ps, pad, shift):
    p = Cache(ns, lens, Hkv, hd, ps, cache, seed=hd + ps)
    Append(p, H, dt, pad=pad, shift=shift, seed=len(ns)).check()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("H,hd", [(0, 64), (4, 32), (4, 128)])
def test_in_place_and_without_queries(dt, cache, H, hd):
    p = Cache([3, 20], [70, 20], 2, hd, 16, cache, seed=1)
    Append(p, H, dt, in_place=H > 0).check()


@pytest.mark.parametrize("dt,cache", TYPES)
def test_positions_and_places_that_are_none(dt, cache):
    """Positions past the tables, before 0, past the page table and in pages outside the pool; rows of nobody at both ends."""
    p = Cache([6, 8, 5], [40, 8, 3], 2, 64, 4, cache, seed=3, extra_table=0, first=2)
    p.table[0, 9] = -1                     # positions 36 .. 39 of sequence 0
    p.table[1, 0] = p.n_pages              # positions 0 .. 3 of sequence 1
    p.lens[1] = 8 + 4 * (p.width - 1)      # its rows reach past the table's width
    for j in range(2, p.width):
        p.table[1, j] = p.table[0, j % 9]
    p.table[1, p.width - 1] = p.table[0, 1]
    Append(p, 4, dt, n_pos=p.lens[1] - 2).check()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("cache", ["e4m3", "e2m1"])
def test_values_that_are_not_finite(dt, cache):
    """Infinities and NaN in q, k and v: NaN in the codes of their head or group alone; sizes near the types' ends."""
    p = Cache([12], [15], 1, 128, 8, cache, seed=4)
    x = torch.randn((16, 4 * 128), generator=torch.Generator().manual_seed(5))
    x[1, 7] = x[2, 200] = float("inf")
    x[3, 130] = x[4, 400] = float("nan")
    x[5] *= 1e38
    x[6] *= 1e-38
    x[7] = 0
    x[8, 128:] = -0.0
    a = Append(p, 2, dt, x=x.cuda())
    if cache == "e2m1":
        a.check()
        return
    # NaN codes of either sign
    out, pools = a.expect()
    call("aic_hip_kv_append", *a.args(), stream())
    for name in "kv":
        got, want = p.pool[name][0].cpu(), pools[name][0]
        nan = (want & 127) == 127
        assert torch.equal((got & 127) == 127, nan) and torch.equal(got[~nan], want[~nan])
        assert torch.equal(p.pool[name][1].cpu(), pools[name][1])


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "e2m1")])
def test_as_rope_and_write(dt, cache):
    """Against the separate calls, one sequence: the rotation off by its two roundings at most."""
    p = Cache([50], [50], 2, 64, 16, cache, seed=6)
    a = Append(p, 4, dt, tail=0)
    x = a.x.clone()
    call("aic_hip_rope", ptr(x), a.ld, 1, 50, 6, 64, 0, ptr(a.dev_c), ptr(a.dev_s), 0, CODE[dt], stream())
    call("aic_hip_kv_append", *a.args(), stream())
    got, want = a.out[:, :256].double(), x[:, :256].double()
    size = a.x[:, :256].double().view(50, 4, 2, 32).norm(dim=2).repeat(1, 1, 2).view(50, 256)
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}[dt]
    # each is off by three fp32 roundings of numbers up to `size` and one of the type's
    assert ((got - want).abs() <= 2 * (3 * 2.0 ** -24 * size + half * want.abs()) * 1.01).all()


def test_captured_on_another_stream():
    p = Cache([1, 1, 30], [100, 7, 60], 2, 128, 16, "e2m1", seed=8)
    a = Append(p, 4, "bf16")
    out, pools = a.expect()
    args = a.args()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call("aic_hip_kv_append", *args, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        _filled(p)
        a.out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.out.cpu(), out)
        for name in "kv":
            for g, e in zip(p.pool[name], pools[name]):
                assert torch.equal(g.cpu(), e)
