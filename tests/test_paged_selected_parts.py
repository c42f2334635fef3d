"""Which calls of attention over chosen pages divide their rows' keys among blocks, by the workspace that they ask for (no GPU needed): rows may
be of any lengths, so long ones are not left to a block each for being many."""
import pytest

from autonomousaicore_amd import _lib
from autonomousaicore_amd._lib import AIC_BF16, AIC_U4, AIC_U8
from tests.test_paged_refusals import P, cache

CODES = dict(k_exps=P, v_exps=P)


@pytest.mark.parametrize("kw", [dict(type=AIC_BF16), dict(type=AIC_U8, **CODES), dict(type=AIC_U4, **CODES)])
@pytest.mark.parametrize("rows", [1, 16, 27, 28, 32, 48, 64, 128, 255])
@pytest.mark.parametrize("pages", [129, 512, 4096])
def test_long_rows_are_divided(kw, rows, pages):
    size = _lib.load().aic_hip_attn_paged_selected_workspace
    c = cache(page_size=64, kv_heads=8, head_dim=128, **kw)
    assert size(c, rows, pages, 32) > 0


@pytest.mark.parametrize("rows,pages,whole", [(1, 16, True), (1, 17, False), (16, 64, True), (16, 65, False), (28, 128, True), (32, 128, True),
                                              (48, 17, False), (64, 128, True), (256, 4096, True)])
def test_what_a_block_takes_whole(rows, pages, whole):
    size = _lib.load().aic_hip_attn_paged_selected_workspace
    assert (size(cache(page_size=64, kv_heads=8, head_dim=128), rows, pages, 32) == 0) == whole
