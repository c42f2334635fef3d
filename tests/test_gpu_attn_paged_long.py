"""Attention of single fp32 tokens over long undivided caches (csrc/kernels/attention_paged_f32_few.hip): no error that
grows with the number of keys times the scores."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from tests.gpu_util import call, host, ptr, stream  # noqa: E402
from tests.paged_ref import CODE, Paged, e4m3_decode, e4m3_encode  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def _shared(B, n, L, hd, cache, k, v):
    """B sequences of n rows over one cache of L tokens, k and v [L, hd] exact in it; so many that no keys are divided."""
    ps = 64
    p = Paged([n], [L], 1, hd, ps, cache, seed=3)
    pages = p.table[0, :L // ps]
    for name, x in (("k", k), ("v", v)):
        pool = np.zeros((p.n_pages, 1, ps, hd))
        pool[pages, 0] = x.reshape(-1, ps, hd)
        if cache == "e4m3":
            codes, exps = e4m3_encode(pool)
            assert (e4m3_decode(codes, exps) == pool).all()
            p.pool[name] = torch.from_numpy(codes).cuda(), torch.from_numpy(exps).cuda()
        else:
            p.pool[name] = torch.from_numpy(pool).float().cuda(), None
    p.B, p.ns, p.lens = B, [n] * B, [L] * B
    p.offs, p.table = [n * b for b in range(B + 1)], np.repeat(p.table, B, 0)
    return p


def _attend(p, q, scale):
    """(o, lse) in 64 bits' type of fp32 queries q [B n, hd]."""
    rows, n, hd = len(q), p.ns[0], p.hd
    dq, o, lse = torch.from_numpy(q).float().cuda(), torch.zeros((rows, hd), device="cuda"), torch.zeros(rows, device="cuda")
    c = p.struct()
    call("aic_hip_attn_paged", c, ptr(dq), hd, ptr(o), hd, ptr(lse), ptr(p.dev_offs), ptr(p.dev_lens), p.B, rows, n, p.lens[0], 1, 0,
         scale, None, 0, CODE["f32"], stream())
    return host(o).astype(np.float64), host(lse).astype(np.float64)


@pytest.mark.parametrize("cache", ["f32", "e4m3"])
@pytest.mark.parametrize("hd,L,n", [(32, 65536, 1), (32, 65536, 3), (128, 16384, 1), (128, 65536, 1), (64, 65536, 2)])
def test_weights_keep_their_size_over_a_long_cache(cache, hd, L, n):
    """512 sequences share one cache, so that no keys are divided.  Every product and score is exact in fp32, the scores lie
    near 60, and the largest returns with each batch of keys, so the running maximum soon stands still.  v is positive
    in the first half and negative in the second: a factor that each batch brings to the older weights shows.

    Bounds, relative to sum p |v|: a lane group adds its L / (4 * 256 / hd) keys one by one.  Each addition to o is off by half
    a step of the sum so far, which is at most half of all there is (2^-25), each one to l by up to 2^-24; o, which is
    nearly 0 here, takes l's error times itself.  The joins of groups and waves, exp2 and the rounding of a weight's argument
    add 16 half steps, and the rounding of maximum * c (|m c| < 128: 2^-18) counts twice where two groups' maxima differ."""
    B, j = 512, np.arange(L)
    k, v = np.zeros((L, hd)), np.empty((L, hd))
    k[:, 0], k[:, 1] = 4.0, -((j * hd // 256) % 8) / 2.0
    v[:] = np.where(j < L // 2, 1.0, -1.0)[:, None] * (1 + (np.arange(hd) % 4) / 4.0)
    p = _shared(B, n, L, hd, cache, k, v)
    rows, scale = B * n, 0.25
    q = np.zeros((rows, hd))
    q[:, 0] = 58 + (np.arange(rows) % 64) / 16.0  # scores of 58 to 62
    q[:, 1] = 1 + np.arange(rows) % 3
    o, lse = _attend(p, q, scale)
    # the last row of a sequence sees all keys, the ones before it one less each
    pos = L - n + np.arange(rows) % n
    s = scale * np.outer(q[:192 * n, 1], k[:, 1])  # the first component is the same for all keys; rows repeat after 192
    w = np.exp(s) * (j[None] <= pos[:192 * n, None])
    tot = w.sum(1, keepdims=True)
    ref, ab = (w / tot) @ v, (w / tot) @ np.abs(v)
    ref_lse = scale * 4.0 * q[:, 0] + np.log(tot[np.arange(rows) % (192 * n), 0])
    ref, ab = ref[np.arange(rows) % (192 * n)], ab[np.arange(rows) % (192 * n)]
    adds = L / (4 * 256 / hd)
    off = np.abs(o - ref) / ab
    tol = (adds / 2 + 16) * 2.0 ** -24 + 2 * 2.0 ** -18 * math.log(2) + adds * 2.0 ** -24 * np.abs(ref) / ab
    assert not (off > tol).any() and np.isfinite(off).all(), (float(off.max()), float(tol.max()))
    # log2's argument, the maximum's product and the three roundings after it, of values below 128 and 64
    off, tol = np.abs(lse - ref_lse), (adds + 16) * 2.0 ** -24 + 3 * 2.0 ** -18 * math.log(2) + 62 * 2.0 ** -22
    assert off.max() <= tol, (float(off.max()), tol)


@pytest.mark.parametrize("cache", ["f32", "e4m3"])
@pytest.mark.parametrize("hd,L,n", [(32, 131072, 1), (64, 131072, 4), (128, 131072, 1), (128, 65536, 2)])
def test_small_weights_are_not_lost_one_by_one(cache, hd, L, n):
    """One key of weight 1 for each lane group, then only keys of weight e^-17.5 = 2^-25.2: each by itself is less than half a step
    of the sum.  Added up by batches of 8 they are not.

    Bound, relative to sum p |v|: L / (32 * 256 / hd) batches for a lane group, each addition off by half a step of the sum so
    far, to l and to o; the 8 weights of a batch and the joins of groups and waves 24 half steps more; a weight's argument is
    25 with two roundings and the rounding of log2 e, 75 * 2^-24 in all and log 2 times that in the weight."""
    B, j = 512, np.arange(L)
    big = (j < 4 * 2048 // hd) & ((j * hd // 256) % 8 == 0)
    k, v = np.zeros((L, hd)), np.ones((L, hd))
    k[~big, 1], v[big] = -64.0, 0.0
    p = _shared(B, n, L, hd, cache, k, v)
    q = np.zeros((B * n, hd))
    q[:, 1] = 1.0
    scale = 17.5 / 64
    o, lse = _attend(p, q, scale)
    seen = L - n + np.arange(B * n) % n + 1
    small = (seen - big.sum()) * math.exp(-17.5)
    tot = big.sum() + small
    batches = L / (32 * 256 / hd)
    tol = 2 * (batches + 24) * 2.0 ** -24 + 75 * 2.0 ** -24
    off = np.abs(o / (small / tot)[:, None] - 1)
    assert off.max() <= tol, (float(off.max()), tol)
    off = np.abs(lse - np.log(tot))
    assert off.max() <= tol, (float(off.max()), tol)
