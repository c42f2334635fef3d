"""The ends of an e4m3 cache's range: finite numbers stay finite when they are read, in the cache's operators and in attention
over it.  The largest number that fp32 and bf16 share with the codes is 240 * 2^120; 256 * 2^120 is 2^128."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from tests.gpu_util import call, ptr, stream  # noqa: E402
from tests.paged_ref import CODE, TORCH, Paged, e4m3_decode, e4m3_encode  # noqa: E402
from tests.test_gpu_attn_paged import Call  # noqa: E402
from tests.test_gpu_attn_paged_range import FORMS, _check  # noqa: E402

TOP = 240.0 * 2.0 ** 120


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def _values(codes, exps):
    with np.errstate(over="ignore"):
        return np.clip(e4m3_decode(codes, exps), -TOP, TOP)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_rows_at_the_ends_read_back(dt, hd):
    """Written and read: the nearest code, and the largest one in the range for what would be past it."""
    big, rng = torch.finfo(TORCH[dt]).max, np.random.default_rng(hd)
    rows = np.zeros((9, hd))
    rows[0, [1, 5]] = big, -big
    rows[1] = np.linspace(-3.39e38, 3.39e38, hd)
    rows[2, :4] = 247 * 2.0 ** 120, 248 * 2.0 ** 120, 249 * 2.0 ** 120, -240 * 2.0 ** 120
    rows[3] = 2.98e38
    rows[4] = 2.0 ** -133 * (np.arange(hd) - 20)      # subnormal
    rows[5] = 2.0 ** -118 * rng.standard_normal(hd)   # codes' subnormals below bf16's least number
    rows[6, :3] = np.inf, -np.inf, big                # held as NaN beside the finite one
    rows[7, 0] = np.nan
    rows[8] = rng.standard_normal(hd)
    n = len(rows)
    p = Paged([n], [n], 1, hd, 4, "e4m3", seed=2)
    x = torch.from_numpy(np.concatenate([rows, -rows], 1)).to(TORCH[dt]).cuda()
    y = torch.zeros_like(x)
    args = (2 * hd, None, None, 1, n, CODE[dt], stream())
    for name, t in (("aic_hip_kv_write", x), ("aic_hip_kv_read", y)):
        c = p.struct()
        call(name, c, ptr(t), ptr(t) + hd * t.element_size(), args[0], ptr(p.dev_offs), ptr(p.dev_lens), *args[3:])
    torch.cuda.synchronize()
    got, ref = y.cpu(), x.double().cpu().numpy()
    for i in range(2):
        want = torch.from_numpy(_values(*e4m3_encode(ref[:, i * hd:(i + 1) * hd]))).to(TORCH[dt])
        mine = got[:, i * hd:(i + 1) * hd]
        assert torch.equal(mine.isnan(), want.isnan())
        assert torch.equal(mine.nan_to_num(7.0), want.nan_to_num(7.0))
        assert torch.isfinite(mine).numpy()[np.isfinite(ref[:, i * hd:(i + 1) * hd])].all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("which", ["v", "k"])
@pytest.mark.parametrize("byte", [247, 250, 254])
@pytest.mark.parametrize("n,L,H,Hkv,hd", FORMS)
def test_attention_over_rows_at_the_top(dt, which, byte, n, L, H, Hkv, hd):
    """A fifth of the rows with the largest powers, whose larger codes are past the range, others of 2^113 or of 1 beside them."""
    p = Paged([n], [L], Hkv, hd, 16, "e4m3", seed=n + L)
    rng = np.random.default_rng(byte)
    codes, exps = (t.cpu().numpy() for t in p.pool[which])
    u = rng.random(exps.shape)
    exps = np.where(u < 0.2, byte, np.where(u < 0.3, 240, exps)).astype(np.uint8)
    p.pool[which] = torch.from_numpy(codes).cuda(), torch.from_numpy(exps).cuda()
    setattr(p, which, _values(codes, exps))
    q = np.random.default_rng(n).standard_normal((n + 3, H * hd))
    # keys up to 2^128: queries that leave the scores at a few units
    _check(Call(p, H, dt, q=torch.from_numpy(q * 2.0 ** -125 if which == "k" else q)).run(), dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,L", [(1, 300), (40, 300), (200, 200)])
def test_a_window_of_one_gives_the_row_itself(dt, n, L):
    """(w v) (1 / w) with the one weight w = 2^d, d the rounding of its argument: three roundings by at most 2^-24 each, below
    2^-22 together, which bf16's rounding takes off again."""
    p = Paged([n], [L], 1, 64, 16, "e4m3", seed=n)
    codes, exps = p.pool["v"]
    exps.fill_(247)
    p.v = _values(codes.cpu().numpy(), exps.cpu().numpy())
    a = Call(p, 1, dt, window=1).run()
    torch.cuda.synchronize()
    want = torch.from_numpy(p.rows("v", 0, 0)[L - n:]).to(TORCH[dt])
    got = a.o[:n, :64].cpu()
    assert torch.equal(got, want) if dt == "bf16" else ((got.double() - want.double()).abs() <= want.double().abs() * 2.0 ** -22).all()
