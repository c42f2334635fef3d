"""Sizes of the calls over the paged key/value cache at the ends of their types: refused, in the size queries too, with nothing
computed from them (no GPU needed)."""
import pytest

from autonomousaicore_amd import _lib
from autonomousaicore_amd._lib import AIC_BF16, AIC_F16, AIC_U8

from tests.test_paged_refusals import DTYPE, INVALID, OUT_OF_RANGE, P, SHAPE, cache, refused

HUGE = [1 << 31, 1 << 40, (1 << 62), (1 << 63) - 1]


def attention(c, q=P, o=2 * P, ld=1 << 20, H=4, T=1, max_len=9, n=0, max_q=1):
    return (c, q, ld, o, ld, None, P, P, 1, T, max_q, max_len, H, 0, 0.125, None, n, AIC_BF16, None)


@pytest.mark.parametrize("H", HUGE)
@pytest.mark.parametrize("T", [1, 2, 1 << 20])
def test_heads(H, T):
    """H * head_dim and T * H / kv_heads do not wrap around."""
    c = cache(kv_heads=1)
    with pytest.raises(_lib.AicError) as e:
        _lib.call("aic_hip_attn_paged", *attention(c, ld=(1 << 63) - 1, H=H, T=T))
    assert e.value.code in (INVALID, OUT_OF_RANGE)
    assert _lib.load().aic_hip_attn_paged_workspace(c, 1, T, 1, 9, H) in (-INVALID, -OUT_OF_RANGE)


@pytest.mark.parametrize("kw,code", [(dict(head_dim=-2), INVALID), (dict(head_dim=0), INVALID), (dict(head_dim=48), INVALID), (dict(head_dim=1 << 62), INVALID),
                                     (dict(kv_heads=4097), INVALID), (dict(kv_heads=-1), SHAPE), (dict(kv_heads=0), SHAPE), (dict(type=AIC_F16), DTYPE)])
def test_size_queries_refuse_what_the_call_refuses(kw, code):
    c = cache(**kw)
    H = kw.get("kv_heads", 2) * 2
    for max_len in (9, 600, 100000):
        assert _lib.load().aic_hip_attn_paged_workspace(c, 4, 8, 2, max_len, H) == -code
    refused(code, "head|cache", "aic_hip_attn_paged", *attention(c, H=H))


def test_cache_sizes_of_rows():
    """kv_heads * head_dim does not wrap around on its way to the leading dimension's check."""
    for kw in (dict(kv_heads=1 << 57, head_dim=128), dict(kv_heads=(1 << 62), head_dim=64, type=AIC_U8)):
        for name in ("aic_hip_kv_write", "aic_hip_kv_read"):
            refused(INVALID, "kv_heads|exps", name, cache(**kw), P, P, 1 << 20, P, P, 1, 1, AIC_BF16, None)


def test_a_query_size_without_a_place_for_the_cache():
    """The size is asked before the pools are there."""
    c = cache(k_pages=None, v_pages=None, page_table=None)
    assert _lib.load().aic_hip_attn_paged_workspace(c, 1, 1, 1, 100000, 4) > 0


def test_output_in_the_place_of_the_queries():
    refused(INVALID, "overlap", "aic_hip_attn_paged", *attention(cache(), o=P))
