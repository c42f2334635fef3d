"""What the further calls over the paged key/value cache refuse: an error code and a message before anything is launched (no GPU
needed)."""
import pytest

from autonomousaicore_amd import _lib
from autonomousaicore_amd._lib import AIC_BF16, AIC_F16, AIC_F32, AIC_U4, AIC_U8
from tests.test_paged_refusals import DTYPE, INVALID, OUT_OF_RANGE, P, SHAPE, cache, refused

HUGE = [1 << 31, 1 << 40, 1 << 62, (1 << 63) - 1]


def codes(**kw):
    return cache(**{**dict(type=AIC_U4, k_exps=P, v_exps=P), **kw})


def append(c=None, **kw):
    a = {**dict(q=P, ld_q=256, out=2 * P, ld_o=256, H=4, k=P, v=P, ld=128, cos=P, sin=P, n_pos=9, offs=P, lens=P, B=2, T=4, dt=AIC_BF16), **kw}
    return (c or cache(), *[a[k] for k in ("q", "ld_q", "out", "ld_o", "H", "k", "v", "ld", "cos", "sin", "n_pos", "offs", "lens", "B", "T", "dt")], None)


def bounds(c=None, **kw):
    a = {**dict(bounds=P, offs=P, lens=P, B=2, T=4), **kw}
    return (c or cache(), a["bounds"], a["offs"], a["lens"], a["B"], a["T"], None)


def select(c=None, **kw):
    a = {**dict(bounds=P, q=P, ld=256, offs=P, lens=P, B=2, T=4, max_q=2, max_len=900, H=4, first=1, last=2, n=8, picked=P, plens=P, ws=P,
                size=1 << 30, dt=AIC_BF16), **kw}
    return (c or cache(), *[a[k] for k in ("bounds", "q", "ld", "offs", "lens", "B", "T", "max_q", "max_len", "H", "first", "last", "n", "picked",
                                           "plens", "ws", "size", "dt")], None)


def chosen(c=None, **kw):
    a = {**dict(q=P, ld_q=256, o=2 * P, ld_o=256, lse=None, picked=P, plens=P, T=4, n=8, H=4, scale=0.1, ws=P, size=1 << 30, dt=AIC_BF16), **kw}
    return (c or cache(), *[a[k] for k in ("q", "ld_q", "o", "ld_o", "lse", "picked", "plens", "T", "n", "H", "scale", "ws", "size", "dt")], None)


CALLS = [("aic_hip_kv_append", append), ("aic_hip_kv_bounds", bounds), ("aic_hip_kv_select", select), ("aic_hip_attn_paged_selected", chosen)]
BAD_CACHES = [(dict(type=AIC_F16), DTYPE, "cache"), (dict(head_dim=48), INVALID, "head_dim"), (dict(head_dim=-64), INVALID, "head_dim"),
              (dict(kv_heads=0), INVALID, "heads"), (dict(kv_heads=4097), INVALID, "heads"), (dict(page_size=0), INVALID, "page_size"),
              (dict(page_size=65537), INVALID, "page_size"), (dict(n_pages=0), INVALID, "n_pages"), (dict(n_pages=1 << 31), INVALID, "n_pages"),
              (dict(k_pages=None), INVALID, "null"), (dict(v_pages=P + 8), INVALID, "aligned"), (dict(type=AIC_U8), INVALID, "exps"),
              (dict(type=AIC_U4), INVALID, "exps"), (dict(type=AIC_U4, k_exps=P, v_exps=P + 2), INVALID, "4-byte")]


@pytest.mark.parametrize("kw,code,words", BAD_CACHES)
@pytest.mark.parametrize("name,args", CALLS)
def test_caches(name, args, kw, code, words):
    refused(code, words, name, *args(cache(**kw)))


@pytest.mark.parametrize("name", ["aic_hip_kv_write", "aic_hip_kv_read", "aic_hip_attn_paged"])
def test_codes_of_four_bits(name):
    """The calls that were there take the type and look at its exponents."""
    for kw in (dict(k_exps=None), dict(v_exps=None), dict(k_exps=P + 1)):
        c = codes(**kw)
        args = (c, P, 4096, 2 * P, 4096, None, P, P, 1, 1, 1, 1, 4, 0, 0.125, None, 0, AIC_BF16, None) if "attn" in name else (
            c, P, P, 1 << 20, P, P, 1, 1, AIC_BF16, None)
        refused(INVALID, "exps|exponents", name, *args)
    size = _lib.load().aic_hip_attn_paged_workspace
    assert size(codes(), 1, 1, 1, 100000, 4) > 0 and size(codes(), 1, 1, 1, 100, 4) >= 0


@pytest.mark.parametrize("name,args", CALLS)
def test_nothing_to_do(name, args):
    _lib.call(name, *args(T=0, **(dict(q=None, o=None, picked=None, plens=None) if args is chosen else {})))
    refused(INVALID, "descriptor", name, None, *args()[1:])


def test_append():
    name = "aic_hip_kv_append"
    for k in ("q", "out", "k", "v", "cos", "sin", "offs", "lens"):
        refused(INVALID, "null", name, *append(**{k: None}))
    refused(INVALID, "leading", name, *append(ld=127))
    refused(INVALID, "leading", name, *append(ld_q=255))
    refused(INVALID, "leading", name, *append(ld_o=255))
    refused(INVALID, "leading", name, *append(out=P, ld_o=264))  # in place, other rows
    refused(INVALID, "H must", name, *append(H=-1))
    refused(INVALID, "H must", name, *append(H=65537, ld_q=1 << 40, ld_o=1 << 40))
    refused(INVALID, "n_pos", name, *append(n_pos=0))
    refused(INVALID, "B and T", name, *append(B=-1))
    refused(INVALID, "B and T", name, *append(T=1 << 31))
    refused(DTYPE, "rows", name, *append(dt=AIC_F16))
    refused(DTYPE, "cache", name, *append(dt=AIC_F32))
    refused(DTYPE, "rows", name, *append(codes(), dt=AIC_U4))
    for h in HUGE:
        refused(INVALID, "H must", name, *append(H=h))


def test_bounds():
    name = "aic_hip_kv_bounds"
    for k in ("bounds", "offs", "lens"):
        refused(INVALID, "null", name, *bounds(**{k: None}))
    refused(INVALID, "aligned", name, *bounds(bounds=P + 8))
    refused(INVALID, "B and T", name, *bounds(B=-1))
    refused(INVALID, "B and T", name, *bounds(T=-1))


def test_select():
    name = "aic_hip_kv_select"
    for k in ("bounds", "q", "offs", "lens", "picked", "plens"):
        refused(INVALID, "null", name, *select(**{k: None}))
    refused(INVALID, "aligned", name, *select(bounds=P + 8))
    refused(INVALID, "leading", name, *select(ld=255))
    refused(SHAPE, "heads", name, *select(H=3))
    refused(SHAPE, "heads", name, *select(H=0))
    refused(INVALID, "B must", name, *select(B=-1))
    refused(INVALID, "T must", name, *select(T=-1))
    refused(INVALID, "max_q", name, *select(max_q=-1))
    refused(INVALID, "max_len", name, *select(max_len=-1))
    refused(INVALID, "max_len", name, *select(max_len=1 << 31))
    for kw in (dict(first=-1), dict(last=0), dict(n=2), dict(n=0), dict(n=(1 << 24) + 1), dict(first=(1 << 63) - 1), dict(last=(1 << 63) - 1)):
        refused(INVALID, "n_sel", name, *select(**kw))
    refused(DTYPE, "queries", name, *select(dt=AIC_F16))
    refused(DTYPE, "cache", name, *select(dt=AIC_F32))
    size = _lib.load().aic_hip_kv_select_workspace
    n = size(cache(), 4, 900)
    assert n == 4 * 2 * 57 * 8 and size(cache(), 0, 900) == 0
    refused(INVALID, "workspace", name, *select(size=n - 1))
    refused(INVALID, "workspace", name, *select(size=-1))
    refused(INVALID, "workspace", name, *select(ws=P + 8))
    assert size(cache(page_size=0), 4, 900) == -INVALID and size(None, 4, 900) == -INVALID
    assert size(cache(page_size=1, kv_heads=4096), (1 << 31) - 1, (1 << 31) - 4096) == -OUT_OF_RANGE
    for h in HUGE:
        refused(INVALID, "query heads|H", name, *select(H=h if h % 2 == 0 else h - 1, ld=(1 << 63) - 1))


def test_chosen():
    name = "aic_hip_attn_paged_selected"
    for k in ("q", "o", "picked", "plens"):
        refused(INVALID, "null", name, *chosen(**{k: None}))
    refused(INVALID, "overlap", name, *chosen(o=P))
    refused(INVALID, "leading", name, *chosen(ld_q=255))
    refused(INVALID, "leading", name, *chosen(ld_o=255))
    refused(SHAPE, "heads", name, *chosen(H=3))
    refused(INVALID, "T must", name, *chosen(T=-1))
    refused(INVALID, "n_sel", name, *chosen(n=0))
    refused(INVALID, "n_sel", name, *chosen(n=1 << 27))  # of 16 positions each
    refused(INVALID, "scale", name, *chosen(scale=0.0))
    refused(INVALID, "scale", name, *chosen(scale=float("nan")))
    refused(DTYPE, "queries", name, *chosen(dt=AIC_F16))
    refused(DTYPE, "cache", name, *chosen(dt=AIC_F32))
    refused(OUT_OF_RANGE, "rows", name, *chosen(T=1 << 30))
    size = _lib.load().aic_hip_attn_paged_selected_workspace
    n = size(cache(), 1, 1000, 4)
    assert n > 0 and size(cache(), 1, 4, 4) == 0 and size(cache(), 0, 4, 4) == 0
    refused(INVALID, "workspace", name, *chosen(T=1, n=1000, size=n - 1))
    refused(INVALID, "workspace", name, *chosen(T=1, n=1000, size=-1))
    refused(INVALID, "workspace", name, *chosen(T=1, n=1000, ws=P + 8))
    assert size(cache(), 1, 0, 4) == -INVALID and size(cache(), 1, 4, 3) == -SHAPE and size(None, 1, 4, 4) == -INVALID
    for h in HUGE:
        with pytest.raises(_lib.AicError) as e:
            _lib.call(name, *chosen(H=h if h % 2 == 0 else h - 1, ld_q=(1 << 63) - 1, ld_o=(1 << 63) - 1))
        assert e.value.code in (INVALID, OUT_OF_RANGE)
