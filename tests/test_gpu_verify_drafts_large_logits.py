"""Verification of drafted tokens on logits far from zero (csrc/kernels/drafts.hip): the sums of both distributions keep
their digits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from tests.test_gpu_verify_drafts import Batch  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


@pytest.mark.parametrize("temperature,base,step", [(1.0, 2.0 ** 22, 0.5), (0.0011, 2.0 ** 13, 0.0009765625), (0.25, -2.0 ** 20, 0.125)])
def test_a_residual_of_one_token_far_from_zero(temperature, base, step):
    """The target's distribution is even but for one token, the draft's but for another of the same weight: only the first is
    left of p - d, and a uniform next to 1 draws it.  The target's logits lie around `base`, the draft's around zero: a
    relative error e of a row's sum would leave V e over the other tokens, which the last 2^-24 of the whole shows from e = 1e-11 on."""
    V, B = 4096, 16
    b = Batch([2] * B, V, "f32", temperature, seed=1)
    b.z, b.y = torch.zeros(b.T, V, dtype=torch.float32), torch.zeros(b.T, V, dtype=torch.float32)
    b.u[:], b.u_next[:] = 0.999, 1.0 - 2.0 ** -24
    for s in range(B):
        b.z[2 * s:2 * s + 2] = base + np.sign(base) * s * 64 * step
        b.z[2 * s, 5 + s] += step
        b.y[2 * s, 3000 + s] += step
        b.ids[2 * s + 1] = 3000 + s
    assert (b.z[::2, 5:5 + B].amax(1) - b.z[::2, 100])[:B].eq(step).all()
    b.device().launch().check()
    assert (b.counts == 1).all() and b.tokens[:, 0].tolist() == [5 + s for s in range(B)]
