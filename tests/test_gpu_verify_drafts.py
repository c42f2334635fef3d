"""Verification of drafted tokens (csrc/kernels/drafts.hip) against its definition in 64 bits: every token, count and length
equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests import paged_ref  # noqa: E402
from tests.gpu_util import call, ptr, stream  # noqa: E402

CODE, TORCH = paged_ref.CODE, paged_ref.TORCH


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


class Batch:
    def __init__(self, ns, V, dt, temperature, one_hot=False, pad=0, shift=0, seed=0, first=0, max_q=None, near=0.7):
        self.ns, self.V, self.dt, self.temperature, self.B = ns, V, dt, temperature, len(ns)
        rng = np.random.default_rng(seed)
        self.offs = [first + sum(ns[:b]) for b in range(self.B + 1)]
        self.T, self.ld, self.shift = self.offs[-1] + 2, V + pad, shift
        self.max_q = max(max(ns), 1) if max_q is None else max_q
        z = rng.standard_normal((self.T, V)) * 2.5
        self.z = torch.from_numpy(z).to(TORCH[dt])
        self.y = None if one_hot else torch.from_numpy(z + near * rng.standard_normal((self.T, V))).to(TORCH[dt])
        self.lens = [int(n) + int(x) for n, x in zip(ns, rng.integers(1, 99, self.B))]
        self.u, self.u_next = rng.random(self.T).astype(np.float32), rng.random(self.B).astype(np.float32)
        # drafts: draws from the draft's distribution, as a drafting model's
        w = (self.y if self.y is not None else self.z).double().numpy() / max(temperature, 0.05)
        w = np.exp(w - w.max(1, keepdims=True))
        run = np.cumsum(w, 1)
        at = (run < run[:, -1:] * rng.random((self.T, 1))).sum(1)
        self.ids = np.concatenate([[0], np.minimum(at[:-1], V - 1)]).astype(np.int64)

    def _rows(self, x):
        buf = torch.full((self.T * self.ld + self.shift + 16,), float("nan"), dtype=TORCH[self.dt], device="cuda")
        view = buf[self.shift:self.shift + self.T * self.ld].view(self.T, self.ld)
        view[:, :self.V] = x.cuda()
        return buf, view

    def device(self):
        d = lambda a: torch.as_tensor(a).cuda()  # noqa: E731
        self.keep = self._rows(self.z), None if self.y is None else self._rows(self.y)
        self.d = dict(ids=d(self.ids), u=d(self.u), u_next=d(self.u_next), offs=d(np.array(self.offs, np.int64)),
                      lens=d(np.array(self.lens, np.int64)))
        self.tokens = torch.full((self.B, self.max_q), 77, dtype=torch.int64, device="cuda")
        self.counts, self.new = (torch.full((self.B,), 77, dtype=torch.int64, device="cuda") for _ in range(2))
        return self

    def launch(self, ws=None, st=None, new=True):
        z, y, d = self.keep[0][1], self.keep[1], self.d
        call("aic_hip_verify_drafts", ptr(z), self.ld, None if y is None else ptr(y[1]), self.ld, ptr(d["ids"]), ptr(d["u"]),
             ptr(d["u_next"]), ptr(d["offs"]), ptr(d["lens"]), self.B, self.T, self.max_q, self.V, self.temperature, ptr(self.tokens),
             ptr(self.counts), ptr(self.new) if new else None, ptr(ws), 0 if ws is None else ws.numel(), CODE[self.dt],
             stream() if st is None else st)
        return self

    def expect(self):
        y = None if self.y is None else self.y.double().numpy()
        return paged_ref.drafts(self.z.double().numpy(), y, self.ids, self.u, self.u_next, self.offs, self.lens, self.max_q, self.V,
                                self.temperature)

    def check(self, want=None):
        torch.cuda.synchronize()
        for got, exp in zip((self.tokens, self.counts, self.new), self.expect() if want is None else want):
            assert np.array_equal(got.cpu().numpy(), exp)
        return self


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("one_hot", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.001, 0.0011, 0.7, 1.0, 20.0])
@pytest.mark.parametrize("ns,V,pad,shift", [([1], 1, 0, 0), ([5, 1, 0, 3], 2, 3, 0), ([4, 8, 1, 2], 1000, 0, 0), ([3, 0, 5], 4096, 8, 1),
                                            ([6, 2], 4097, 0, 0), ([5, 5, 1], 32000, 0, 0)])
def test_tokens_counts_and_lengths(dt, one_hot, temperature, ns, V, pad, shift):
    Batch(ns, V, dt, temperature, one_hot, pad, shift, seed=V + len(ns)).device().launch().check()


def test_long_drafts_and_rows_before_the_first():
    Batch([300, 1, 40], 130, "f32", 1.0, seed=3, first=4, near=0.1).device().launch().check()


def test_rows_past_max_q_are_not_looked_at():
    Batch([6, 2, 5], 500, "f32", 1.0, seed=4, max_q=3, near=0.05).device().launch().check()


def test_a_draft_from_the_same_distribution_is_kept():
    b = Batch([8, 8], 999, "f32", 0.8, seed=5, near=0.0)
    b.u[:] = np.float32(1.0 - 2.0 ** -24)
    b.device().launch().check()
    assert (b.counts == 8).all()


def test_uniforms_at_their_ends():
    for u, v in ((0.0, 0.0), (0.0, 1.0 - 2.0 ** -24), (1.0 - 2.0 ** -24, 0.0), (1.0 - 2.0 ** -24, 1.0 - 2.0 ** -24)):
        b = Batch([3, 3, 1], 5000, "f32", 1.0, seed=6, near=3.0)
        b.u[:], b.u_next[:] = u, v
        b.device().launch().check()


def test_uniforms_outside_their_range_give_tokens_of_the_row():
    """At and past 1, and NaN: no draft is kept by a NaN, and the last token of any weight is drawn."""
    for v in (1.0, 3.0, float("nan")):
        b = Batch([3, 1], 700, "f32", 1.0, seed=7)
        b.u[:], b.u_next[:] = np.nan, v
        b.device().launch()
        torch.cuda.synchronize()
        assert (b.counts == 1).all() and ((b.tokens[:, 0] >= 0) & (b.tokens[:, 0] < 700)).all()


@pytest.mark.parametrize("one_hot", [False, True])
def test_drafts_that_are_no_tokens(one_hot):
    b = Batch([4, 4, 4], 300, "f32", 1.0, one_hot, seed=8)
    b.ids[1], b.ids[6], b.ids[9] = -1, 300, 2 ** 40
    b.device().launch().check()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_infinities_and_nan_among_the_logits(dt, temperature):
    b = Batch([3, 2, 2, 1, 1, 2], 5000, dt, temperature, seed=9)
    z = b.z
    z[0, ::2] = float("-inf")                       # half of the vocabulary is shut out
    z[1, 17:4500] = float("nan")                    # NaN counts as shut out
    z[3, [40, 4000]] = float("inf")                 # the mass is shared by the infinities
    z[4] = float("-inf")
    z[5, :4999] = float("-inf")                     # one token left
    z[7] = float("nan")                             # nothing to draw: -1
    z[8, 4096:] = float("-inf")                     # a whole part shut out
    b.y[9, 100:] = float("nan")
    b.y[0, 3:] = float("-inf")
    b.device().launch().check()


def test_equal_logits_go_to_the_lowest_index():
    b = Batch([2, 1, 1], 9000, "bf16", 0.0, seed=10)
    b.z[:] = b.z.clamp(max=1.0)
    b.device().launch().check()


def test_workspaces_capture_and_lengths_in_place():
    b = Batch([5, 3, 1], 32000, "f32", 0.8, seed=11).device()
    n = _lib.load().aic_hip_verify_drafts_workspace(b.B, b.T, b.V)
    ws = torch.full((n,), 0xff, dtype=torch.uint8, device="cuda")
    with pytest.raises(_lib.AicError, match="workspace"):
        b.launch(ws[:n - 16])
    b.launch(ws).check()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        with pytest.raises(_lib.AicError, match="captured"):
            b.launch(None, s.cuda_stream)
        b.launch(ws, s.cuda_stream)
    for turn in range(3):
        c = Batch([5, 3, 1], 32000, "f32", 0.8, seed=20 + turn).device()
        b.keep[0][1].copy_(c.keep[0][1])
        b.keep[1][1].copy_(c.keep[1][1])
        for k in b.d:
            b.d[k].copy_(c.d[k])
        b.tokens.fill_(5)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        c.launch()  # eager, on another stream
        b.check(c.check().expect())
    want = b.new.clone()
    call("aic_hip_verify_drafts", ptr(b.keep[0][1]), b.ld, ptr(b.keep[1][1]), b.ld, ptr(b.d["ids"]), ptr(b.d["u"]), ptr(b.d["u_next"]),
         ptr(b.d["offs"]), ptr(b.d["lens"]), b.B, b.T, b.max_q, b.V, b.temperature, ptr(b.tokens), ptr(b.counts), ptr(b.d["lens"]), None, 0,
         CODE["f32"], stream())
    torch.cuda.synchronize()
    assert torch.equal(b.d["lens"], want)


def test_no_rows_at_all():
    b = Batch([0, 0], 10, "f32", 1.0, seed=1).device().launch().check()
    assert (b.tokens == -1).all() and (b.counts == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1e30, 1e36, 3e38])
def test_temperatures_up_to_the_largest(dt, temperature):
    """Nearly equal weights of all logits but the shut out ones."""
    b = Batch([3, 2, 1], 3000, dt, temperature, seed=11)
    b.z[:, 5:2900] = float("-inf")
    b.z[1, 7] = float("nan")
    b.device().launch().check()


@pytest.mark.parametrize("u", [0.9375, 1.0])
def test_a_residual_that_is_nothing_in_64_bits(u):
    """p and d differ at one token of weight 1e-26 alone, which no sum holds: the new token is p's."""
    b = Batch([2, 2], 3000, "f32", 1.0, seed=12, near=0.0)
    for row, seq in ((0, 0), (2, 1)):
        b.z[row, 40], b.y[row, 40] = -61.0, -60.0
        b.ids[row + 1] = 40
    b.u[:] = u
    b.device().launch().check()
    assert (b.counts == 1).all() and (b.tokens[:, 0] >= 0).all()
