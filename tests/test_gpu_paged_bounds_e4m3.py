"""Bounds of e4m3 pages whose values are below bf16's least number: rounded outwards, so that they hold every key."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from tests.paged_codes_ref import Cache, bounds  # noqa: E402
from tests.paged_ref import e4m3_decode  # noqa: E402
from tests.test_gpu_paged_select import _run_bounds  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


@pytest.mark.parametrize("hd,ps", [(32, 1), (64, 3), (128, 16)])
@pytest.mark.parametrize("top", [3, 20, 127])
def test_bounds_below_the_least_number(hd, ps, top):
    p = Cache([7, 40], [30, 90], 2, hd, ps, "e4m3", seed=hd)
    rng = np.random.default_rng(ps + top)
    shape = (p.n_pages, 2, ps, hd)
    codes = rng.integers(0, top, shape) | rng.integers(0, 2, shape) << 7  # 127 would be no number
    exps = rng.integers(1, 4, shape[:-1])
    codes[0, 0, 0, 5] = 127
    p.pool["k"] = torch.from_numpy(codes.astype(np.uint8)).cuda(), torch.from_numpy(exps.astype(np.uint8)).cuda()
    p.k = e4m3_decode(codes, exps)
    out = torch.full((p.n_pages, 2, 2, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    before = out.cpu().double().numpy()
    want = bounds(p, before)
    touched = want != before
    steps = want * 2.0 ** 133  # bf16's numbers up to 2^-125 are whole ones; all others here are held
    want = np.where(touched, np.stack([np.floor(steps[:, :, 0]), np.ceil(steps[:, :, 1])], 2) * 2.0 ** -133, want)
    _run_bounds(p, out)
    got = out.cpu().double().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    assert top > 100 or (want[touched] != bounds(p, before)[touched]).any()
