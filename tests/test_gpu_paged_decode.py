"""The paged cache's operators together, as a serving loop runs them: prompts of different lengths, then drafted tokens
written, attended and verified, the lengths going on from what was kept.  Greedy verification gives exactly the tokens of
greedy decoding without drafts, whatever the drafts were: checked against a one-layer model recomputed from the whole
sequence in 64 bits for every token."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests.gpu_util import call, ptr, stream  # noqa: E402
from tests.paged_ref import CODE, TORCH, e4m3_decode, e4m3_encode  # noqa: E402

V, D, H, HKV, HD, PS = 97, 96, 4, 2, 32, 5


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


class Model:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        g = lambda *s: rng.standard_normal(s) / math.sqrt(s[0])  # noqa: E731
        self.E, self.Wqkv, self.Wo = rng.standard_normal((V, D)), g(D, (H + 2 * HKV) * HD) * 2, g(H * HD, D) * 3
        self.dev = [torch.from_numpy(x).float().cuda() for x in (self.E, self.Wqkv, self.Wo)]

    def next_token(self, ids, cache):
        """Greedy next token after ids, in float64."""
        x = self.E[ids]
        qkv = (x @ self.Wqkv).astype(np.float32).astype(np.float64)
        q = qkv[-1, :H * HD].reshape(H, HD)
        k, v = (qkv[:, (H + i * HKV) * HD:(H + (i + 1) * HKV) * HD].reshape(-1, HKV, HD) for i in range(2))
        if cache == "e4m3":
            k, v = (e4m3_decode(*e4m3_encode(t)) for t in (k, v))
        out = []
        for h in range(H):
            s = k[:, h * HKV // H] @ q[h] / math.sqrt(HD)
            w = np.exp(s - s.max())
            out.append((w / w.sum()) @ v[:, h * HKV // H])
        z = (x[-1] + np.concatenate(out) @ self.Wo) @ self.E.T
        top = np.sort(z)[-2:]
        assert top[1] - top[0] > 1e-3, "the test's seed gives a tie"
        return int(z.argmax())


class Serving:
    def __init__(self, model, B, pages, cache):
        self.m, self.B = model, B
        pool = (pages, HKV, PS, HD)
        self.pools = [torch.full(pool, 0xff, dtype=torch.uint8, device="cuda") if cache == "e4m3" else
                      torch.full(pool, float("nan"), dtype=TORCH[cache], device="cuda") for _ in range(2)]
        self.exps = [torch.zeros(pool[:3], dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.table = torch.from_numpy(np.random.default_rng(0).permutation(pages).reshape(B, -1).astype(np.int32)).cuda()
        e = self.exps if cache == "e4m3" else [None, None]
        self.c = _lib.KVPages(ptr(self.pools[0]), ptr(self.pools[1]), ptr(e[0]), ptr(e[1]), ptr(self.table), self.table.shape[1], pages, PS, HKV, HD,
                              CODE[cache])

    def step(self, chunks, cached):
        """The chunks' rows written and attended; their logits.  cached: tokens in the cache before them."""
        ns = [len(c) for c in chunks]
        self.offs = torch.tensor([sum(ns[:b]) for b in range(self.B + 1)], device="cuda")
        self.lens = torch.tensor([c + n for c, n in zip(cached, ns)], device="cuda")
        self.ids = torch.tensor([t for c in chunks for t in c], device="cuda")
        T, c, w = sum(ns), ctypes.byref(self.c), H * HD
        E, Wqkv, Wo = self.m.dev
        x = E[self.ids]
        qkv = (x.double() @ Wqkv.double()).float()
        ld, batch = qkv.shape[1], (ptr(self.offs), ptr(self.lens), self.B, T)
        call("aic_hip_kv_write", c, ptr(qkv) + w * 4, ptr(qkv) + (w + HKV * HD) * 4, ld, *batch, CODE["f32"], stream())
        o = torch.empty((T, w), device="cuda")
        call("aic_hip_attn_paged", c, ptr(qkv), ld, ptr(o), w, None, *batch, max(ns), max(x + n for x, n in zip(cached, ns)), H, 0,
             1 / math.sqrt(HD), None, 0, CODE["f32"], stream())
        return ((x.double() + o.double() @ Wo.double()) @ E.double().t()).float().contiguous()

    def verify(self, logits, ids, offs, lens, max_q):
        tokens = torch.empty((self.B, max_q), dtype=torch.int64, device="cuda")
        counts, new = (torch.empty(self.B, dtype=torch.int64, device="cuda") for _ in range(2))
        call("aic_hip_verify_drafts", ptr(logits), V, None, 0, ptr(ids), None, None, ptr(offs), ptr(lens), self.B,
             logits.shape[0], max_q, V, 0.0, ptr(tokens), ptr(counts), ptr(new), None, 0, CODE["f32"], stream())
        counts = counts.tolist()
        return [t[:n] for t, n in zip(tokens.tolist(), counts)], new.tolist()


@pytest.mark.parametrize("cache", ["f32", "e4m3"])
def test_speculative_decoding_gives_the_greedy_tokens(cache):
    rng = np.random.default_rng(7)
    m = Model(3)
    prompts = [rng.integers(0, V, n).tolist() for n in (1, 23, 9)]
    s = Serving(m, 3, 3 * 20, cache)
    logits = s.step(prompts, [0, 0, 0])
    last = (s.offs[1:] - 1)
    one = torch.arange(4, device="cuda")
    got, cached = s.verify(logits[last].contiguous(), s.ids[last], one, s.lens, 1)
    text = [p + g for p, g in zip(prompts, got)]
    kept = drafted = 0
    while min(len(t) - len(p) for t, p in zip(text, prompts)) < 40:
        chunks = []
        for b, t in enumerate(text):
            assert cached[b] == len(t) - 1  # all but the newest token are in the cache
            draft, ids = [], list(t)
            for _ in range(int(rng.integers(0, 6)) if len(t) < 90 else 0):  # right ones, and wrong ones now and then
                nxt = m.next_token(ids, cache)
                draft.append(nxt if rng.random() < 0.75 else int(rng.integers(0, V)))
                ids.append(draft[-1])
            chunks.append([t[-1]] + draft)
        logits = s.step(chunks, cached)
        got, cached = s.verify(logits, s.ids, s.offs, s.lens, max(len(c) for c in chunks))
        for b in range(3):
            drafted += len(chunks[b]) - 1
            kept += len(got[b]) - 1
            text[b] = text[b] + got[b]
    assert 0 < kept < drafted
    for p, t in zip(prompts, text):
        for i in range(len(p), len(t)):
            assert t[i] == m.next_token(t[:i], cache), (i, len(p))
    # the cache reads back as what the kept tokens wrote
    n = [len(t) - 1 for t in text]
    offs, lens = torch.tensor([0] + np.cumsum(n).tolist(), device="cuda"), torch.tensor(n, device="cuda")
    k, v = (torch.empty((sum(n), HKV * HD), device="cuda") for _ in range(2))
    call("aic_hip_kv_read", ctypes.byref(s.c), ptr(k), ptr(v), HKV * HD, ptr(offs), ptr(lens), 3, sum(n), CODE["f32"], stream())
    qkv = (m.dev[0][torch.tensor([x for t in text for x in t[:-1]], device="cuda")].double() @ m.dev[1].double()).float().cpu().numpy().astype(np.float64)
    for i, x in enumerate((k, v)):
        want = qkv[:, (H + i * HKV) * HD:(H + (i + 1) * HKV) * HD].reshape(-1, HKV, HD)
        want = e4m3_decode(*e4m3_encode(want)) if cache == "e4m3" else want
        assert np.array_equal(x.cpu().numpy().astype(np.float64), want.reshape(x.shape))
