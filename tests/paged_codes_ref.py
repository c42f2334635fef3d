"""The paged cache's further forms for the tests, from their definitions in numpy: 4-bit codes with a power of two per 32
elements, the rotation on the way into the cache, the bounds of pages, and the choice of pages by them."""
import ctypes

import numpy as np
import torch

from autonomousaicore_amd import _lib
from tests.paged_ref import CODE, TORCH, Paged, e4m3_encode

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
CACHE_CODE = {**CODE, "e2m1": _lib.AIC_U4}


def e2m1_encode(x):
    """float64 rows [..., hd] -> (bytes of two codes, exponent bytes [..., hd / 32]): nearest code, ties to the even one."""
    x = np.asarray(x, np.float64).reshape(x.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    top = np.abs(x).max(-1)
    m, e = np.frexp(top)                       # top = m 2^e, 0.5 <= m < 1; 6 = 0.75 2^3
    e = np.where(m <= 0.75, e - 3, e - 2)
    e = np.where(top > 0, np.clip(e, -126, 125), 0)
    y = np.minimum(np.abs(x) * 2.0 ** -e[..., None].astype(np.float64), 6.0)
    hi = np.clip(np.searchsorted(VALUES, y), 0, 7)
    lo = np.maximum(hi - 1, 0)
    dl, dh = y - VALUES[lo], VALUES[hi] - y
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(x) & ~bad[..., None], code | 8, code).astype(np.uint8)
    code = code.reshape(code.shape[:-2] + (-1,))
    return code[..., 0::2] | code[..., 1::2] << 4, np.where(bad, 255, e + 127).astype(np.uint8)


def e2m1_decode(codes, exps):
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1, 32))
    v = np.where(c & 8, -VALUES[c & 7], VALUES[c & 7]) * 2.0 ** (exps.astype(np.float64) - 127)[..., None]
    return np.where(exps[..., None] == 255, np.nan, v).reshape(codes.shape[:-1] + (-1,))


class Cache(Paged):
    """Paged, with 4-bit pools too."""

    def __init__(self, ns, lens, Hkv, hd, ps, cache, seed=0, extra_table=2, first=0):
        super().__init__(ns, lens, Hkv, hd, ps, "f32" if cache == "e2m1" else cache, seed, extra_table, first)
        if cache == "e2m1":
            for name in "kv":
                self.set_codes(name, *e2m1_encode(getattr(self, name)))
        self.cache = cache

    def set_codes(self, name, codes, exps):
        self.pool[name] = torch.from_numpy(codes).cuda(), torch.from_numpy(exps).cuda()
        setattr(self, name, e2m1_decode(codes, exps))

    def struct(self):
        if self.cache != "e2m1":
            return super().struct()
        self.cache = "e4m3"  # pointers and sizes are laid out alike
        super().struct()
        self.cache = "e2m1"
        self.c.type = _lib.AIC_U4
        return ctypes.byref(self.c)


def encode(rows, cache):
    """float64 rows -> what a cache of codes holds of them."""
    return e2m1_encode(rows) if cache == "e2m1" else e4m3_encode(rows)


def turn(x, c, s):
    """Rows [n, heads, hd] (fp32) turned by [n, hd / 2] tables, operation by operation in fp32."""
    with np.errstate(all="ignore"):
        x1, x2 = np.split(x.astype(np.float32), 2, -1)
        c, s = c[:, None].astype(np.float32), s[:, None].astype(np.float32)
        return np.concatenate([x1 * c - x2 * s, x1 * s + x2 * c], -1)


def bounds(p, before):
    """What kv_bounds leaves where `before` [n_pages, Hkv, 2, hd] stood."""
    out = before.copy()
    for b in range(p.B):
        n, L = p.ns[b], p.lens[b]
        if n == 0 or L <= 0:
            continue
        for pi in range(max(L - n, 0) // p.ps, (L - 1) // p.ps + 1):
            at = p.place(b, pi * p.ps)
            if at is None:
                continue
            keys = p.k[at[0], :, :min(p.ps, L - pi * p.ps)]
            out[at[0], :, 0], out[at[0], :, 1] = keys.min(1), keys.max(1)  # numpy's keep a NaN
    return out


def select(p, bound, q, H, first, last, n_sel, max_len):
    """(picked, lens) from float64 bounds and queries [T, H, hd]."""
    T = q.shape[0]
    picked, lens = np.full((T, p.Hkv, n_sel), -1, np.int32), np.full((T, p.Hkv), -1, np.int64)
    G = H // p.Hkv
    for b in range(p.B):
        for i in range(p.ns[b]):
            t, pos = p.offs[b] + i, p.lens[b] - p.ns[b] + i
            P = pos // p.ps + 1 if pos >= 0 else 0
            lens[t] = pos + 1 if pos >= 0 else 0
            if P > -(-max_len // p.ps):
                lens[t] = 1
                continue
            ids = [int(p.table[b, j]) if j < p.width else -1 for j in range(P)]
            for h in range(p.Hkv):
                take = np.arange(P)
                if P > n_sel:
                    score = np.full(P, np.inf)
                    for j, page in enumerate(ids):
                        if 0 <= page < p.n_pages:
                            with np.errstate(all="ignore"):
                                x = q[t, h * G:(h + 1) * G]
                                s = np.where(x >= 0, x * bound[page, h, 1], x * bound[page, h, 0]).sum(-1).max()
                            score[j] = np.inf if np.isnan(s) else s
                    free = np.arange(first, P - last)
                    best = free[np.argsort(-score[free], kind="stable")[:n_sel - first - last]]
                    take = np.sort(np.concatenate([np.arange(first), best, np.arange(P - last, P)]))
                    lens[t, h] = (n_sel - 1) * p.ps + pos % p.ps + 1
                picked[t, h, :len(take)] = np.array(ids, np.int64)[take].astype(np.int32)
    return picked, lens
