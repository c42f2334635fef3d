"""The choice of pages needs no workspace where every row takes all its pages: captured, with none and with a small one."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from autonomousaicore_amd import _lib  # noqa: E402
from tests.gpu_util import call, host  # noqa: E402
from tests.paged_codes_ref import Cache  # noqa: E402
from tests.test_gpu_paged_select import Choice  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.set_device(0)


def _captured(a, args):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call("aic_hip_kv_select", *args, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        a.picked.fill_(77), a.lens.fill_(77)
        graph.replay()
        torch.cuda.synchronize()
        yield


@pytest.mark.parametrize("pages", [7, 600, 2100])  # pages of a thread that chooses: 2, 8 and any number
def test_all_pages_captured_without_a_workspace(pages):
    ps = 4
    p = Cache([2, 1, 0], [ps * pages, 3, 5], 2, 32, ps, "bf16", seed=pages)
    a = Choice(p, 4, "bf16", 1, 2, pages)
    want = a.want()
    args = a.args()
    held = p.dev_table, p.dev_offs, p.dev_lens
    for _ in _captured(a, args):
        assert np.array_equal(host(a.lens), want[1]) and np.array_equal(host(a.picked), want[0])
    del held
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    a.run(small).check()


def test_no_sequences_captured_without_a_workspace():
    p = Cache([1], [900], 2, 32, 4, "bf16", seed=1)
    a = Choice(p, 4, "bf16", 1, 2, 8)
    args = list(a.args())
    args[6] = 0  # B
    for _ in _captured(a, args):
        assert (host(a.picked) == -1).all() and (host(a.lens) == -1).all()


def test_one_page_more_needs_it():
    p = Cache([2, 1], [33, 3], 2, 32, 4, "bf16", seed=1)
    a = Choice(p, 4, "bf16", 1, 2, 8)  # of nine
    with pytest.raises(_lib.AicError, match="workspace"):
        a.run(torch.empty(a.bytes() - 16, dtype=torch.uint8, device="cuda"))
    args = a.args()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.lens.fill_(77)
        with pytest.raises(_lib.AicError, match="captured"):
            call("aic_hip_kv_select", *args, torch.cuda.current_stream().cuda_stream)
    a.run().check()
