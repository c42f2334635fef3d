"""What the calls over the paged key/value cache refuse: an error code and a message before anything is launched (no GPU
needed)."""
import ctypes as C

import pytest

import autonomousaicore_amd as aic
from autonomousaicore_amd import _lib
from autonomousaicore_amd._lib import AIC_BF16, AIC_F16, AIC_F32, AIC_U8

P = 1 << 20  # a 16-byte aligned address that is never followed
INVALID, OUT_OF_RANGE, SHAPE, DTYPE = 1, 2, 3, 4


def cache(**kw):
    c = _lib.KVPages(P, P, None, None, P, 8, 100, 16, 2, 64, AIC_BF16)
    for k, v in kw.items():
        setattr(c, k, v)
    return C.byref(c)


def refused(code, words, name, *args):
    with pytest.raises(aic.AicError, match=words) as e:
        _lib.call(name, *args)
    assert e.value.code == code, e.value


BAD_CACHES = [(dict(type=AIC_F16), DTYPE, "cache"), (dict(head_dim=48), INVALID, "head_dim"), (dict(head_dim=256), INVALID, "head_dim"),
              (dict(kv_heads=0), INVALID, "kv_heads|heads"), (dict(page_size=0), INVALID, "page_size"),
              (dict(page_size=65537), INVALID, "page_size"), (dict(n_pages=0), INVALID, "n_pages"), (dict(n_pages=1 << 31), INVALID, "n_pages"),
              (dict(ld_table=0), INVALID, "ld_table"), (dict(k_pages=None), INVALID, "null"), (dict(page_table=None), INVALID, "null"),
              (dict(v_pages=P + 8), INVALID, "aligned"), (dict(type=AIC_U8), INVALID, "exps"), (dict(type=AIC_F32), DTYPE, "cache")]


@pytest.mark.parametrize("kw,code,words", BAD_CACHES)
def test_caches(kw, code, words):
    for name in ("aic_hip_kv_write", "aic_hip_kv_read"):
        if kw.get("kv_heads") != 0:
            refused(code, words, name, cache(**kw), P, P, 1 << 20, P, P, 1, 1, AIC_BF16, None)
    if kw.get("kv_heads") == 0:
        code, words = SHAPE, "heads"
    refused(code, words, "aic_hip_attn_paged", cache(**kw), P, 4096, P, 4096, None, P, P, 1, 1, 1, 1, 4, 0, 0.125, None, 0, AIC_BF16, None)


@pytest.mark.parametrize("name", ["aic_hip_kv_write", "aic_hip_kv_read"])
def test_rows(name):
    ok = dict(k=P, v=P, ld=128, offs=P, lens=P, B=2, T=4, dt=AIC_BF16)

    def bad(code, words, **kw):
        a = {**ok, **kw}
        refused(code, words, name, cache(), a["k"], a["v"], a["ld"], a["offs"], a["lens"], a["B"], a["T"], a["dt"], None)

    bad(INVALID, "leading", ld=127)
    bad(INVALID, "null", k=None)
    bad(INVALID, "null", offs=None)
    bad(INVALID, "null", lens=None)
    bad(INVALID, "B and T", B=-1)
    bad(INVALID, "B and T", T=1 << 31)
    bad(DTYPE, "rows", dt=AIC_F16)
    bad(DTYPE, "cache", dt=AIC_F32)
    refused(INVALID, "descriptor", name, None, P, P, 128, P, P, 1, 1, AIC_BF16, None)
    _lib.call(name, cache(), None, None, 128, None, None, 0, 0, AIC_BF16, None)  # nothing to do


def test_attention():
    ok = dict(q=P, ld_q=256, o=P, ld_o=256, offs=P, lens=P, B=2, T=4, max_q=2, max_len=9, H=4, window=0, scale=0.1, ws=None, n=0, dt=AIC_BF16)

    def bad(code, words, c=None, **kw):
        a = {**ok, **kw}
        refused(code, words, "aic_hip_attn_paged", c or cache(), a["q"], a["ld_q"], a["o"], a["ld_o"], None, a["offs"], a["lens"], a["B"], a["T"],
                a["max_q"], a["max_len"], a["H"], a["window"], a["scale"], a["ws"], a["n"], a["dt"], None)

    bad(INVALID, "leading", ld_q=255)
    bad(INVALID, "leading", ld_o=255)
    bad(INVALID, "null", q=None)
    bad(INVALID, "null", o=None)
    bad(INVALID, "null", lens=None)
    bad(SHAPE, "heads", H=3)
    bad(SHAPE, "heads", H=0)
    bad(INVALID, "scale", scale=0.0)
    bad(INVALID, "scale", scale=float("nan"))
    bad(INVALID, "scale", scale=float("inf"))
    bad(INVALID, "scale", scale=3e38)  # infinite in units of log 2
    bad(INVALID, "window", window=-1)
    bad(INVALID, "max_len", max_len=1 << 31)
    bad(INVALID, "max_q", max_q=-1)
    bad(INVALID, "workspace", n=-1)
    bad(OUT_OF_RANGE, "rows", T=1 << 30)
    bad(DTYPE, "queries", dt=AIC_F16)
    bad(DTYPE, "cache", dt=AIC_F32)
    size = _lib.load().aic_hip_attn_paged_workspace
    n = size(cache(), 1, 1, 1, 100000, 4)
    assert n > 0 and size(cache(), 1, 1, 1, 100, 4) == 0 and size(cache(), 0, 0, 0, 0, 4) == 0
    bad(INVALID, "workspace", B=1, T=1, max_q=1, max_len=100000, ws=P, n=n - 1)
    bad(INVALID, "workspace", B=1, T=1, max_q=1, max_len=100000, ws=P + 8, n=n)
    assert size(cache(), 1, 1, 1, 100, 3) == -SHAPE and size(None, 1, 1, 1, 1, 1) == -INVALID
    _lib.call("aic_hip_attn_paged", cache(), None, 256, None, 256, None, None, None, 0, 0, 0, 0, 4, 0, 0.1, None, 0, AIC_BF16, None)


def test_drafts():
    ok = dict(z=P, ld=50, y=P, ldy=50, ids=P, u=P, un=P, offs=P, lens=P, B=2, T=4, max_q=2, V=50, temp=1.0, tok=P, cnt=P, new=P, ws=P,
              n=1 << 20, dt=AIC_F32)

    def bad(code, words, **kw):
        a = {**ok, **kw}
        refused(code, words, "aic_hip_verify_drafts", *[a[k] for k in ("z", "ld", "y", "ldy", "ids", "u", "un", "offs", "lens", "B", "T", "max_q",
                                                                        "V", "temp", "tok", "cnt", "new", "ws", "n", "dt")], None)

    bad(INVALID, "leading", ld=49)
    bad(INVALID, "leading", ldy=49)
    bad(INVALID, "vocabulary", V=0)
    bad(INVALID, "vocabulary", V=(1 << 30) + 1, ld=1 << 31, ldy=1 << 31)
    bad(INVALID, "max_q", max_q=0)
    bad(INVALID, "temperature", temp=-0.5)
    bad(INVALID, "temperature", temp=float("nan"))
    bad(INVALID, "null", u=None)
    bad(INVALID, "null", un=None)
    bad(INVALID, "null", ids=None)
    bad(INVALID, "null", z=None)
    bad(INVALID, "null", tok=None)
    bad(INVALID, "null", cnt=None)
    bad(INVALID, "null", lens=None)
    bad(INVALID, "null", offs=None)
    bad(INVALID, "B and T", T=-1)
    bad(DTYPE, "logits", dt=AIC_BF16 + 100)
    bad(INVALID, "workspace", n=10)
    bad(INVALID, "workspace", n=-1)
    bad(INVALID, "workspace", ws=P + 4)
    size = _lib.load().aic_hip_verify_drafts_workspace
    assert size(1, 5, 32000) > 0 and size(-1, 5, 10) == -INVALID
    _lib.call("aic_hip_verify_drafts", None, 50, None, 50, None, None, None, None, None, 0, 0, 1, 50, 1.0, None, None, None, None, 0, AIC_F32, None)
