"""Attention over the paged cache on values near the smallest and the largest numbers, in every form: errors relative to
what is added up, with nothing allowed beside them but fp32's smallest steps."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests.gpu_util import call, host, ptr  # noqa: E402
from tests.paged_ref import CODE, HALF, TORCH, Paged, attention  # noqa: E402
from tests.test_gpu_attn_paged import TYPES, Call  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


# one to a few hundred rows, undivided and divided: (n, L, H, Hkv, hd)
FORMS = [(1, 300, 2, 1, 64), (1, 3000, 2, 2, 128), (1, 300, 8, 1, 32), (3, 2900, 4, 4, 64), (16, 700, 4, 1, 128), (40, 300, 2, 1, 64),
         (40, 2100, 1, 1, 32), (200, 1100, 2, 1, 128), (330, 330, 4, 2, 64)]


def _values(p, x):
    """v of all pages becomes x [n_pages, Hkv, ps, hd] (f32 and bf16 caches)."""
    t = torch.from_numpy(x).to(TORCH[p.cache])
    p.pool["v"], p.v = (t.cuda(), None), t.double().numpy()


def _times(p, by):
    """v times 2^by, exactly."""
    if p.cache == "e4m3":
        p.pool["v"][1].add_(by)
        p.v = p.v * 2.0 ** by
    else:
        _values(p, p.v * 2.0 ** by)


def _check(a, dt):
    """As tests/paged_ref.py's bound: the scores' errors, 2^-18 for a few fp32 steps of weights up to 2^8, half a step for bf16's
    weights and for the output.  Beside it L products and L sums off by half of fp32's smallest step each, on weights whose sum
    is 1 at least."""
    p = a.p
    q = a.q[:, :a.w].double().cpu().numpy().reshape(a.T, a.H, p.hd)
    o, lse, ab, sb = attention(p, q, a.H, a.window, a.scale)
    got, got_lse = host(a.o.contiguous())[:, :a.w].reshape(a.T, a.H, p.hd).astype(np.float64), host(a.lse).astype(np.float64)
    mine = slice(p.offs[0], p.offs[-1])
    o, ab, sb, lse, got, got_lse = o[mine], ab[mine], sb[mine], lse[mine], got[mine], got_lse[mine]
    assert np.isfinite(got).all(), int((~np.isfinite(got)).sum())
    tol = (4 * sb[..., None] + 2.0 ** -18) * ab + HALF[dt] * np.abs(o) * 1.01 + (HALF["bf16"] * ab * 1.01 if dt == "bf16" else 0)
    off = np.abs(got - o) / (tol + max(p.lens) * 2.0 ** -149)
    assert off.max() <= 1, (float(off.max()), np.argwhere(off > 1)[:4].tolist(), int((off > 1).sum()))
    assert (np.abs(got_lse - lse) <= 2 * sb + 2.0 ** -17 + 2.0 ** -22 * np.abs(lse)).all()


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n,L,H,Hkv,hd", FORMS)
@pytest.mark.parametrize("by", [-118, -105, -90])
def test_small_values_keep_their_digits(dt, cache, n, L, H, Hkv, hd, by):
    p = Paged([n], [L], Hkv, hd, 16, cache, seed=n + L)
    if cache == "e4m3":
        by = max(by, -117)  # exponent bytes down to 2
    _times(p, by)
    _check(Call(p, H, dt).run(), dt)


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n,L,H,Hkv,hd", FORMS)
def test_sums_of_large_values_do_not_overflow(dt, cache, n, L, H, Hkv, hd):
    """Values up to 1.9e38 of both signs; then, where the cache holds them, all of one sign and near the largest."""
    p = Paged([n], [L], Hkv, hd, 16, cache, seed=n + L)
    _times(p, 125)
    _check(Call(p, H, dt).run(), dt)
    if cache != "e4m3":
        _values(p, 3e38 + 1e37 * np.clip(p.v * 2.0 ** -125, -3, 3))
        _check(Call(p, H, dt).run(), dt)


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("n,L,H,Hkv,hd", FORMS)
def test_small_values_beside_large_ones(dt, cache, n, L, H, Hkv, hd):
    """Columns of 1e38 beside columns of 2^-110, and sequences of each beside one another."""
    p = Paged([n, n, 2], [L, max(n, L // 2), 90], Hkv, hd, 16, cache, seed=n + L)
    x = p.v * 2.0 ** -110
    x[..., 1::3] = np.where(p.v[..., 1::3] > -0.5, 1e38, -1.5e38)  # sums of one sign
    for j in range(90):  # the last sequence without large columns
        page, slot = p.place(2, j)
        x[page, :, slot] = p.v[page, :, slot] * 2.0 ** -110
    _values(p, x)
    _check(Call(p, H, dt).run(), dt)


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("n,L", [(1, 3000), (3, 2900), (40, 2100)])
def test_large_values_in_some_of_the_parts(dt, cache, n, L):
    """Only a third of the keys is large: the parts that hold none of it are joined with those that do."""
    p = Paged([n], [L], 2, 64, 16, cache, seed=n + L)
    x = p.v * 2.0 ** -100
    for j in range(L // 3, 2 * L // 3):
        page, slot = p.place(0, j)
        x[page, :, slot, ::2] = 2e38
    _values(p, x)
    _check(Call(p, 2, dt).run(), dt)


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n,L", [(1, 900), (5, 2000), (60, 300), (60, 1500)])
def test_large_values_in_rows_of_odd_strides(dt, cache, n, L):
    """Outputs whose rows are not aligned, in a window; nothing else is written by the second pass over the keys."""
    p = Paged([n, 1], [L, 40], 2, 64, 7, cache, seed=n)
    _times(p, 125)
    a = Call(p, 4, dt, window=200, pad=3, shift=1).run()
    _check(a, dt)
    inside = np.zeros(a.buf.numel(), bool)
    inside[a.shift:a.shift + a.T * a.ld].reshape(a.T, a.ld)[p.offs[0]:p.offs[-1], :a.w] = True
    assert np.all(host(a.buf)[~inside] == 7.0) and np.all(host(a.lse)[p.offs[-1]:] == 7.0)


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("n,L", [(1, 300), (1, 2100), (40, 300), (200, 700)])
def test_replays_over_values_that_change_their_size(dt, cache, n, L):
    """One graph over normal, large, normal and small values in turn, between eager calls: each replay equals the eager call bit for
    bit, so no replay leaves anything to the next."""
    p = Paged([n], [L], 2, 64, 16, cache, seed=n + L)
    a, e = Call(p, 4, dt), Call(p, 4, dt)
    ws = [torch.empty(max(a.bytes(), 16), dtype=torch.uint8, device="cuda") for _ in range(2)]
    c = p.struct()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def launch(x, w):
        call("aic_hip_attn_paged", c, ptr(x.q), x.ld, ptr(x.o), x.ld, ptr(x.lse), ptr(p.dev_offs), ptr(p.dev_lens), *x.sizes(), x.H, 0, x.scale,
             ptr(w), w.numel(), CODE[dt], s.cuda_stream)

    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        launch(a, ws[0])
    pool, exps = p.pool["v"]
    normal = pool.clone(), None if exps is None else exps.clone()
    plain = p.v
    for by in (0, 125, 0, -100):
        if exps is None:
            pool.copy_((normal[0].double() * 2.0 ** by).to(pool.dtype))
        else:
            exps.copy_(normal[1].int() + by)
        p.v = plain * 2.0 ** by
        a.buf.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        launch(e, ws[1])
        torch.cuda.synchronize()
        assert torch.equal(a.o, e.o) and torch.equal(a.lse, e.lse)
        _check(a, dt)
    _lib.call("aic_hip_mem_release_stream", s.cuda_stream)
