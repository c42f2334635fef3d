"""A paged key/value cache for the tests: a ragged batch over shuffled pages, and the operators over it
in 64 bits, written from their definitions (numpy; a row at a time where values are not finite)."""
import ctypes
import math

import numpy as np
import torch

from autonomousaicore_amd import _lib

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.uint8}
CODE = {"f32": _lib.AIC_F32, "bf16": _lib.AIC_BF16, "e4m3": _lib.AIC_U8}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}  # half a step of the type, relative


def e4m3_values():
    """The 127 numbers of codes 0 .. 126."""
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)


def e4m3_encode(x):
    """float64 rows [..., hd] -> (codes, exponent bytes): nearest code, ties to the even one; NaN: 0x7f."""
    table = e4m3_values()
    fine = np.isfinite(x)
    top = np.where(fine, np.abs(x), 0).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(top > 0, np.ceil(np.log2(top / 448.0)), 0).astype(np.int64)
    e = np.where(top > 0, np.maximum(e, -126), 0)
    for _ in range(2):  # log2's last bit: the least e that holds top
        e = np.where(top > 448.0 * 2.0 ** e, e + 1, np.where((top > 0) & (e > -126) & (top <= 448.0 * 2.0 ** (e - 1)), e - 1, e))
    y = np.where(fine, np.abs(x), 0) * 2.0 ** -e[..., None].astype(np.float64)
    hi = np.clip(np.searchsorted(table, y), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = y - table[lo], table[hi] - y
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(x), code | 128, code)
    return np.where(fine, code, 0x7f).astype(np.uint8), (e + 127).astype(np.uint8)


def e4m3_decode(codes, exps):
    v = np.append(e4m3_values(), np.nan)[codes & 127]
    return np.where(codes & 128, -v, v) * 2.0 ** (exps.astype(np.float64) - 127)[..., None]


class Paged:
    """Pools with every page's values known on the host (float64 `k`, `v` [n_pages, Hkv, ps, hd]) and a batch
    (ns, lens) over them."""

    def __init__(self, ns, lens, Hkv, hd, ps, cache, seed=0, extra_table=2, first=0):
        self.ns, self.lens, self.Hkv, self.hd, self.ps, self.cache = list(ns), list(lens), Hkv, hd, ps, cache
        rng = np.random.default_rng(seed)
        self.B = len(self.ns)
        self.offs = [first + sum(self.ns[:b]) for b in range(self.B + 1)]
        need = [-(-max(n, 0) // ps) for n in self.lens]
        self.n_pages = sum(need) + 2
        self.width = max(need, default=0) + extra_table
        ids = rng.permutation(self.n_pages)
        # entries past a sequence's pages are garbage that must not be followed
        self.table = np.full((self.B, self.width), 2 ** 31 - 7, np.int32)
        for b in range(self.B):
            at = sum(need[:b])
            self.table[b, :need[b]] = ids[at:at + need[b]]
        shape = (self.n_pages, Hkv, ps, hd)
        self.pool = {}
        for name in "kv":
            x = rng.standard_normal(shape)
            if cache == "e4m3":
                codes, exps = e4m3_encode(x)
                self.pool[name] = torch.from_numpy(codes).cuda(), torch.from_numpy(exps).cuda()
                val = e4m3_decode(codes, exps)
            else:
                t = torch.from_numpy(x).to(TORCH[cache])
                self.pool[name] = t.cuda(), None
                val = t.double().numpy()
            setattr(self, name, val)

    def set_row(self, name, b, pos, h, values):
        """Overwrites one cached row of a sequence (f32 / bf16 caches)."""
        page, slot = self.table[b, pos // self.ps], pos % self.ps
        t = torch.as_tensor(values, dtype=torch.float64).to(TORCH[self.cache])
        self.pool[name][0][page, h, slot] = t.cuda()
        getattr(self, name)[page, h, slot] = t.double().numpy()

    def struct(self):
        self.dev_table = torch.from_numpy(self.table).cuda()
        self.dev_offs = torch.tensor(self.offs, dtype=torch.int64).cuda()
        self.dev_lens = torch.tensor(self.lens, dtype=torch.int64).cuda()
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        (k, ke), (v, ve) = self.pool["k"], self.pool["v"]
        self.c = _lib.KVPages(p(k), p(v), p(ke), p(ve), p(self.dev_table), self.width, self.n_pages, self.ps, self.Hkv,
                              self.hd, CODE[self.cache])
        return ctypes.byref(self.c)

    def place(self, b, pos):
        """(page, slot) or None."""
        if pos < 0 or pos // self.ps >= self.width:
            return None
        page = int(self.table[b, pos // self.ps])
        return (page, pos % self.ps) if 0 <= page < self.n_pages else None

    def rows(self, name, b, h):
        """float64 [len, hd]; NaN where there is no place."""
        out = np.full((max(self.lens[b], 0), self.hd), np.nan)
        for j in range(len(out)):
            at = self.place(b, j)
            if at is not None:
                out[j] = getattr(self, name)[at[0], h, at[1]]
        return out


def attention(p, q, H, window, scale):
    """q: float64 [T, H, hd].  (o, lse, bound_o, bound_s) in 64 bits: bound_s[t, h] bounds how far an fp32 score
    may be off, bound_o[t, h, :] is sum_j p_j |v_j|.  Rows of no sequence: NaN."""
    T = q.shape[0]
    o, lse = np.full((T, H, p.hd), np.nan), np.full((T, H), np.nan)
    ab, sb = np.zeros((T, H, p.hd)), np.zeros((T, H))
    for b in range(p.B):
        for h in range(H):
            g = h * p.Hkv // H
            K, V = p.rows("k", b, g), p.rows("v", b, g)
            n = p.ns[b]
            rows = slice(p.offs[b], p.offs[b] + n)
            if np.isfinite(K).all() and np.isfinite(V).all() and np.isfinite(q[rows, h]).all() and len(K):
                pos, j = p.lens[b] - n + np.arange(n)[:, None], np.arange(len(K))
                seen = (j <= pos) & ((j > pos - window) if window else True)
                s = np.where(seen, scale * (q[rows, h] @ K.T), -np.inf)
                m = s.max(1, keepdims=True)
                w = np.exp(s - np.where(m > -np.inf, m, 0))
                tot = w.sum(1, keepdims=True)
                w = w / np.where(tot > 0, tot, 1)
                o[rows, h], ab[rows, h] = w @ V, w @ np.abs(V)
                with np.errstate(divide="ignore"):
                    lse[rows, h] = (m + np.log(tot))[:, 0]
                sb[rows, h] = scale * np.where(seen, np.abs(q[rows, h]) @ np.abs(K.T), 0).max(1) * (p.hd + 2) * 2.0 ** -24
                continue
            for i in range(p.ns[b]):
                t, pos = p.offs[b] + i, p.lens[b] - p.ns[b] + i
                lo = max(0, pos - window + 1) if window else 0
                if pos < 0:
                    o[t, h], lse[t, h] = 0, -math.inf
                    continue
                with np.errstate(all="ignore"):
                    k, v = K[lo:pos + 1], V[lo:pos + 1]
                    s = scale * (k @ q[t, h])
                    m = s.max()
                    w = np.exp(s - m)
                    tot = w.sum()
                    o[t, h], lse[t, h] = (w / tot) @ v, m if m == -math.inf else m + np.log(tot)
                    ab[t, h] = (w / tot) @ np.abs(v)
                    sb[t, h] = scale * (np.abs(k) @ np.abs(q[t, h])).max() * (p.hd + 2) * 2.0 ** -24
    return o, lse, ab, sb


def check_attention(got, lse, p, q, H, window, scale, dt):
    """Element by element.  The weights' errors: a score off by ds moves a weight and the sum by 2 ds; exp2 and its
    argument, sums over the keys and rescalings are a few fp32 steps of values up to 2^8 of the maximum
    (2^-18 together); bf16 rounds each weight and the output by half a step."""
    o, l, ab, sb = attention(p, q, H, window, scale)
    mine = slice(p.offs[0], p.offs[-1])
    g, r, ab, sb = got.astype(np.float64)[mine], o[mine], ab[mine], sb[mine]
    assert np.array_equal(np.isnan(g), np.isnan(r)), "NaN in other places"
    fine = np.isfinite(r)
    assert np.array_equal(g[~fine & ~np.isnan(r)], r[~fine & ~np.isnan(r)])
    with np.errstate(all="ignore"):
        tol = (4 * sb[..., None] + 2.0 ** -18) * ab + 2 ** -40
        tol = tol + HALF[dt] * np.abs(r) * 1.01 + (HALF["bf16"] * ab * 1.01 if dt == "bf16" else 0)
        off = np.abs(g - r) / tol
    assert not fine.any() or off[fine].max() <= 1, (float(off[fine].max()), np.argwhere(fine & ~(off <= 1))[:4].tolist())
    if lse is not None:
        a, e = lse.astype(np.float64)[mine], l[mine]
        assert np.array_equal(np.isnan(a), np.isnan(e))
        fine = np.isfinite(e)
        assert np.array_equal(a[~fine & ~np.isnan(e)], e[~fine & ~np.isnan(e)])
        assert (np.abs(a[fine] - e[fine]) <= 2 * sb[fine] + 2.0 ** -17 + 2.0 ** -22 * np.abs(e[fine])).all()


def drafts(logits, draft, ids, u, u_next, offs, lens, max_q, V, temperature):
    """Speculative verification, a sequence and a token at a time, in 64 bits."""
    B = len(offs) - 1
    tokens, counts, out = np.full((B, max_q), -1, np.int64), np.zeros(B, np.int64), np.zeros(B, np.int64)
    greedy = temperature <= 0.001

    def dist(z):
        z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
        top = z.max()
        if top == -np.inf:
            return np.zeros(V)
        if greedy:
            return np.eye(1, V, int(z.argmax()))[0]
        with np.errstate(all="ignore"):
            w = np.where(z == top, 1.0, np.exp((z - top) / temperature))
        return w / w.sum()

    for b in range(B):
        n = min(offs[b + 1] - offs[b], max_q)
        out[b] = lens[b] - (offs[b + 1] - offs[b])
        if n == 0:
            continue
        got, left = [], None
        for i in range(n):
            t = offs[b] + i
            p = dist(logits[t])
            if i == n - 1:
                left = p
                break
            x = int(ids[t + 1])
            one = np.zeros(V)
            if 0 <= x < V:
                one[x] = 1.0
            d = one if greedy or draft is None else dist(draft[t])
            px = p[x] if 0 <= x < V else 0.0
            if greedy:
                keep = px == 1.0
            else:
                dx = 1.0 if draft is None else d[x] if 0 <= x < V else 0.0
                keep = float(u[t]) * dx < px
            if keep:
                got.append(x)
            else:
                left = p if greedy else np.maximum(p - d, 0.0)
                break
        if not left.any():  # p - d is nothing in 64 bits: from p
            left = p
        run = np.cumsum(left)
        pos = np.flatnonzero(left > 0)
        if len(pos) == 0:
            new = -1
        elif greedy:
            new = int(pos[0])
        else:
            past = pos[run[pos] > run[-1] * float(u_next[b])]
            new = int(past[0]) if len(past) else int(pos[-1])
        got.append(new)
        tokens[b, :len(got)], counts[b] = got, len(got)
        out[b] += len(got)
    return tokens, counts, out
