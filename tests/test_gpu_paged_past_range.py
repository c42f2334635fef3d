"""Positions past the range that lengths reach (2^31 - 4096) in the calls over the paged key/value cache: no number, not nothing."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from tests.gpu_util import host  # noqa: E402
from tests.paged_codes_ref import Cache  # noqa: E402
from tests.test_gpu_paged_append import TYPES, Append  # noqa: E402
from tests.test_gpu_paged_select import Choice, Picked  # noqa: E402

REACH = 2 ** 31 - 4096


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


# -------------------------------------------------------------------------------------- choice
@pytest.mark.parametrize("max_len", [300, REACH])
@pytest.mark.parametrize("n_sel", [4, 40])
def test_choice_of_sequences_past_the_range(max_len, n_sel):
    """Ids -1 and length 1, as past max_len, so that attention over them is NaN; the other sequences' rows are as they are without them."""
    ps = 16 if max_len == 300 else 65536
    p = Cache([2, 1, 3, 1, 2], [300, 290, 300, 7, 30], 2, 32, 16, "bf16", seed=n_sel)
    p.ps = ps
    a = Choice(p, 4, "bf16", 1, 2, n_sel, max_len=max_len)
    a.run()
    want = host(a.picked).copy(), host(a.lens).copy()
    past = {1: 2 ** 31 - 1, 2: REACH + 1, 3: 2 ** 40}
    for b, n in past.items():
        p.lens[b] = n
        want[0][p.offs[b]:p.offs[b + 1]], want[1][p.offs[b]:p.offs[b + 1]] = -1, 1
    a.picked.fill_(77), a.lens.fill_(77)
    a.run()
    assert np.array_equal(host(a.lens), want[1]) and np.array_equal(host(a.picked), want[0])
    if ps == 16:
        o = Picked(p, 4, "bf16", host(a.picked), host(a.lens)).run().check().o
        assert torch.isnan(o[p.offs[1]:p.offs[4], :128]).all() and not torch.isnan(o[:2, :128]).any()


def test_choice_of_many_rows_past_the_range():
    """A chunk whose last rows are past the range: none of its rows has a choice."""
    p = Cache([40, 40], [900, 900], 2, 64, 16, "bf16", seed=2)
    a = Choice(p, 8, "bf16", 1, 2, 9).run().check()
    want = host(a.picked).copy(), host(a.lens).copy()
    p.lens[0] = REACH + 20
    want[0][:40], want[1][:40] = -1, 1
    a.run()
    assert np.array_equal(host(a.lens), want[1]) and np.array_equal(host(a.picked), want[0])


# ------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dt,cache", TYPES)
@pytest.mark.parametrize("in_place", [False, True])
def test_append_past_the_range(dt, cache, in_place):
    """q is NaN and nothing is written where positions are past 2^31 - 1, as from n_pos on; a chunk that reaches over it; the others as ever."""
    p = Cache([2, 1, 3, 4], [300, 290, 300, 40], 2, 64, 16, cache, seed=3)
    p.lens[1], p.lens[2] = 2 ** 40, 2 ** 31 + 1
    Append(p, 4, dt, n_pos=300, in_place=in_place).check()
