"""Attention over chosen pages where a few rows are long and the others short, at the numbers of rows whose equal lengths need no division."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from tests.paged_codes_ref import Cache  # noqa: E402
from tests.test_gpu_paged_select import TYPES, Picked  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("T,Hkv,G,hd,ps,n_sel", [(28, 8, 2, 32, 64, 130), (65, 8, 1, 32, 128, 65), (112, 2, 4, 64, 32, 257), (300, 2, 1, 64, 100, 82)])
def test_few_long_rows(dt, cache, T, Hkv, G, hd, ps, n_sel):
    p = Cache([1], [ps * (n_sel + 3)], Hkv, hd, ps, cache, seed=T)
    rng = np.random.default_rng(T)
    picked = np.stack([rng.permutation(p.n_pages)[:n_sel] for _ in range(T * Hkv)]).reshape(T, Hkv, n_sel)
    lens = rng.integers(1, 300, (T, Hkv))
    lens[0], lens[T // 2], lens[T - 1] = n_sel * ps, n_sel * ps - 77, 8193
    lens[1], lens[2, 0] = -1, 0
    a = Picked(p, G * Hkv, dt, picked, lens)
    if dt == "bf16":
        assert a.bytes() > 0
    a.run(torch.full((max(a.bytes(), 16),), 0xff, dtype=torch.uint8, device="cuda")).check()
    b = Picked(p, G * Hkv, dt, picked, lens).run()
    assert torch.equal(a.o, b.o) and torch.equal(a.lse, b.lse)
