"""What further operators of serving over a paged key/value cache are measured on.

One pass rotates a ragged batch's queries and keys and appends keys and values to the cache, attends over a
cache held in 4 bits, brings the bounds of the pages up to date, selects pages by them for each query, or
attends over the selected pages.  `run` computes each in plain torch operations, or calls the library where
`own` is true.  Sizes follow the model widths that the library is benchmarked on (12 heads of 64, 16 heads of 128,
4 heads of 32) and grouped key/value heads of them.

A batch is `B` sequences; sequence b brings the rows offsets[b] .. offsets[b + 1] of the packed inputs and its
cache holds lens[b] tokens with them.  Lengths come from the case alone (_shape), the order of the sequences, the
pages' places and all values from the seed.
"""
import ctypes
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.uint8, "e2m1": torch.uint8}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the codes 0 .. 7; 8 more: with the sign
GROUP = 32                                       # neighbouring elements that share a power of two


def listed():
    return [
        # a decode step's tokens of 32 chat sequences, rotated and appended: the smallest call
        dict(name="append_decode_b32", kind="append", B=32, n=1, L=2000, H=16, Hkv=8, hd=128, ps=16, cache="bf16", dtype="bf16"),
        # prompts of up to 2048 tokens at the 1B width, quantised to 4 bits on the way, and read back
        dict(name="append_prompt_e2m1", kind="append", B=8, n=2048, L=2048, H=16, Hkv=8, hd=128, ps=64, cache="e2m1", dtype="bf16"),
        # single-token decoding of one chat sequence at the 125M widths: latency
        dict(name="decode_125m_e2m1_b1", kind="attn", B=1, n=1, L=513, H=12, Hkv=12, hd=64, ps=16, window=0, cache="e2m1", dtype="bf16",
             lse=False),
        # single-token decoding of a batch of long contexts, grouped heads
        dict(name="decode_e2m1_b32", kind="attn", B=32, n=1, L=16384, H=16, Hkv=8, hd=128, ps=64, window=0, cache="e2m1", dtype="bf16",
             lse=False),
        # the target's pass over up to four drafted tokens and the one before them, for 16 sequences, odd pages
        dict(name="verify_e2m1_b16", kind="attn", B=16, n=5, L=3000, H=16, Hkv=16, hd=128, ps=24, window=0, cache="e2m1", dtype="bf16",
             lse=True),
        # a 2048-token chunk of one long prompt behind 6144 cached tokens
        dict(name="chunk_e2m1_2048_of_8192", kind="attn", B=1, n=2048, L=8192, H=16, Hkv=2, hd=128, ps=64, window=0, cache="e2m1",
             dtype="bf16", lse=False),
        # after a decode step of 32 sequences: the one page of each that the step has written to
        dict(name="bounds_decode_b32", kind="bounds", B=32, n=1, L=8000, H=16, Hkv=8, hd=128, ps=64, cache="bf16", dtype="bf16"),
        # after prompts of up to 4096 tokens
        dict(name="bounds_prompt_e2m1", kind="bounds", B=8, n=4096, L=4096, H=16, Hkv=8, hd=128, ps=64, cache="e2m1", dtype="bf16"),
        # 64 of one document's 2048 pages, for one token: latency
        dict(name="select_131k_b1", kind="select", B=1, n=1, L=131000, H=16, Hkv=2, hd=128, ps=64, sel=64, cache="bf16", dtype="bf16"),
        # 64 of up to 512 pages of each of 32 sequences
        dict(name="select_b32", kind="select", B=32, n=1, L=32768, H=16, Hkv=8, hd=128, ps=64, sel=64, cache="bf16", dtype="bf16"),
        # attention over the selected pages, one document
        dict(name="sparse_131k_b1", kind="sparse", B=1, n=1, L=131000, H=16, Hkv=2, hd=128, ps=64, sel=64, cache="e2m1", dtype="bf16",
             lse=False),
        # attention over the selected pages, 32 sequences
        dict(name="sparse_b32", kind="sparse", B=32, n=1, L=32768, H=16, Hkv=8, hd=128, ps=64, sel=64, cache="bf16", dtype="bf16",
             lse=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attn", "attn", "attn", "bounds", "select", "select", "sparse", "sparse"])
    H, hd = rng.choice([(12, 64), (16, 64), (16, 128), (16, 128), (4, 32)])
    G = rng.choice([1, 2, 4] if H < 16 else [1, 2, 8] if hd == 128 else [2, 4, 8])
    case = dict(kind=kind, H=H, Hkv=H // G, hd=hd, ps=rng.choice([16, 16, 24, 32, 64, 64, 128]))
    cache = rng.choice(["e2m1", "e2m1", "e2m1", "bf16", "e4m3", "f32"]) if kind != "attn" else "e2m1"
    dtype = "f32" if cache == "f32" or (cache == "e2m1" and rng.random() < 0.2) else "bf16"
    case.update(cache=cache, dtype=dtype)
    if kind in ("append", "bounds"):
        B = _log(rng, 1, 32)
        n = rng.choice([1, _log(rng, 1, 8192 // B)])
        return dict(case, B=B, n=n, L=n + rng.choice([0, _log(rng, 1, 1000)]))
    if kind == "attn":
        # tokens that come in together: one, a few drafted ones, a chunk of a prompt
        few = 1 if rng.random() < 0.4 else rng.randint(2, 8)
        n = few if rng.random() < 0.6 else _log(rng, 9, 1024)
        B = _log(rng, 1, 30) if n <= 8 else _log(rng, 1, max(1, min(16, 2048 // n)))
        top = 12000 if n <= 8 and dtype != "f32" else 4096 if dtype != "f32" else 1024
        return dict(case, B=B, n=n, L=n + _log(rng, 1, top), window=rng.choice([0, 0, 0, _log(rng, 16, 2000)]), lse=rng.random() < 0.3)
    # pages for each of a few tokens: of short contexts all
    n = 1 if rng.random() < 0.6 else rng.randint(2, 8)
    B = _log(rng, 1, 32 // n)
    case.update(B=B, n=n, L=n + _log(rng, 100, 32000 if dtype != "f32" else 8000), sel=rng.choice([16, 33, 64, _log(rng, 8, 128)]))
    return dict(case, lse=rng.random() < 0.3) if kind == "sparse" else case


# ----------------------------------------------------------------------------------- inputs
FIRST, LAST = 1, 2  # pages that are always selected: the first one, and the row's own with the one before it


def _shape(case):
    """(n_b, len_b) of each sequence, longest first: sequence 0 has the case's n and L, the others
    down to a quarter of them, spread evenly."""
    got = []
    for b in range(case["B"]):
        f = 1.0 if b == 0 else 0.25 + 0.75 * ((b * 0.6180339887498949) % 1.0)
        n = max(1, round(case["n"] * f))
        got.append((n, max(n, round(case["L"] * f))))
    return got


def _pow2(e):
    """2^e in fp32, exactly, for whole e in -126 .. 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x, cache):
    """fp32 [..., hd] -> (codes as bytes, biased exponents): the least power of two that holds the largest value."""
    if cache == "e4m3":
        m, e = torch.frexp(x.abs().amax(-1))
        e = torch.where(m > 0, torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126), torch.zeros_like(e))
        return (x * _pow2(-e).unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)
    x = x.unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0, torch.where(m <= 0.75, e - 3, e - 2).clamp(min=-126, max=125), torch.zeros_like(e))
    y = x * _pow2(-e).unsqueeze(-1)
    a = y.abs()
    # to nearest, ties to the even code
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).byte()
    code = (code + 8 * torch.signbit(y)).byte().flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).to(torch.uint8)


def _dequantise(codes, exps, cache):
    """The fp32 rows that codes and exponents stand for."""
    if cache == "e4m3":
        return codes.view(torch.float8_e4m3fn).float() * _pow2(exps.int() - 127).unsqueeze(-1)
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
    pair = torch.stack([codes & 15, codes >> 4], -1).long()
    x = table[pair].flatten(-2).unflatten(-1, (-1, GROUP))
    return (x * _pow2(exps.int() - 127).unsqueeze(-1)).flatten(-2)


def _pools(case, n_pages):
    """Shapes of a pool and of its exponents (None: none)."""
    at = (n_pages, case["Hkv"], case["ps"])
    if case["cache"] == "e2m1":
        return at + (case["hd"] // 2,), at + (case["hd"] // GROUP,)
    return at + (case["hd"],), at if case["cache"] == "e4m3" else None


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    shape = _shape(case)
    order = torch.randperm(len(shape), generator=g, device="cuda").tolist()
    shape = [shape[i] for i in order]
    ns, lens = [n for n, _ in shape], [n for _, n in shape]
    T, B = sum(ns), len(ns)
    H, Hkv, hd, ps, t, kind, cache = case["H"], case["Hkv"], case["hd"], case["ps"], DT[case["dtype"]], case["kind"], case["cache"]
    pages = [-(-n // ps) for n in lens]
    width, n_pages = max(pages) + 1, sum(pages) + 3
    places = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    for b in range(B):
        at = sum(pages[:b])
        table[b, :pages[b]] = places[at:at + pages[b]]
    s = dict(case=case, B=B, T=T, max_q=max(ns), max_len=max(lens), n_pages=n_pages, table=table, lens=torch.tensor(lens, device="cuda"),
             offsets=torch.tensor([sum(ns[:b]) for b in range(B + 1)], device="cuda"), k_exps=None, v_exps=None)
    pool, exps = _pools(case, n_pages)
    channel = 1.0 + 3.0 * (torch.rand(Hkv, 1, hd, generator=g, device="cuda") > 0.95)  # keys have a few loud channels
    if kind in ("append", "select"):
        # the pool before the call; a selection does not look at it
        for name in "kv":
            s[name + "_pages"] = torch.zeros(pool, dtype=DT[cache], device="cuda")
            s[name + "_exps"] = torch.zeros(exps, dtype=torch.uint8, device="cuda") if exps else None
    else:
        for name in "kv":
            x = randn(n_pages, Hkv, ps, hd)
            x = x * channel if name == "k" else x
            if exps:
                s[name + "_pages"], s[name + "_exps"] = _quantise(x, cache)
            else:
                s[name + "_pages"] = x.to(DT[cache])
            del x
    bounds_t = torch.float32 if cache == "f32" else torch.bfloat16
    if kind == "append":
        s["qkv"] = randn(T, (H + 2 * Hkv) * hd).to(t)
        angle = torch.arange(s["max_len"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q"] = torch.empty(T, H * hd, dtype=t, device="cuda")
        if cache == "e2m1":
            s["back"] = tuple(torch.empty(T, Hkv * hd, dtype=t, device="cuda") for _ in range(2))
    elif kind == "bounds":
        s["bounds"] = torch.zeros(n_pages, Hkv, 2, hd, dtype=bounds_t, device="cuda")
    else:
        s["q_in"] = (randn(T, H * hd) * 1.5).to(t)
    if kind == "select":
        middle, reach = randn(n_pages, Hkv, hd) * 0.4 * channel[:, 0], (1.5 + 0.4 * randn(n_pages, Hkv, hd).abs()) * channel[:, 0]
        s["bounds"] = torch.stack([middle - reach, middle + reach], 2).to(bounds_t)
        s["picked"] = torch.empty(T, Hkv, case["sel"], dtype=torch.int32, device="cuda")
        s["picked_lens"] = torch.empty(T, Hkv, dtype=torch.int64, device="cuda")
    if kind == "sparse":
        # the first page, the last two, and others of the row's, by a score of another layer
        b, pos = _rows(s)
        s["picked"], s["picked_lens"] = _pick(s, torch.rand(T, Hkv, width, generator=g, device="cuda", dtype=torch.float64), b, pos)
    if kind in ("attn", "sparse"):
        s["o"] = torch.empty(T, H * hd, dtype=t, device="cuda")
        s["lse"] = torch.empty(T, H, device="cuda") if case["lse"] else None
    if own:
        _handle(s)
    return s


# ------------------------------------------------------------------------ the library's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _handle(s):
    """The cache's descriptor and the workspace, as a serving program keeps them."""
    from autonomousaicore_amd import _lib
    case = s["case"]
    code = {"f32": _lib.AIC_F32, "bf16": _lib.AIC_BF16, "e4m3": _lib.AIC_U8, "e2m1": _lib.AIC_U4}
    s["cache"] = _lib.KVPages(_ptr(s["k_pages"]), _ptr(s["v_pages"]), _ptr(s["k_exps"]), _ptr(s["v_exps"]), _ptr(s["table"]),
                              s["table"].shape[1], s["n_pages"], case["ps"], case["Hkv"], case["hd"], code[case["cache"]])
    s["dt"] = code[case["dtype"]]
    lib, cache, n = _lib.load(), ctypes.byref(s["cache"]), 0
    if case["kind"] == "attn":
        n = lib.aic_hip_attn_paged_workspace(cache, s["B"], s["T"], s["max_q"], s["max_len"], case["H"])
    elif case["kind"] == "select":
        n = lib.aic_hip_kv_select_workspace(cache, s["T"], s["max_len"])
    elif case["kind"] == "sparse":
        n = lib.aic_hip_attn_paged_selected_workspace(cache, s["T"], case["sel"], case["H"])
    s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")


def _run_own(s):
    from autonomousaicore_amd import _lib
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    H, Hkv, hd, kind = case["H"], case["Hkv"], case["hd"], case["kind"]
    cache, batch = ctypes.byref(s["cache"]), (_ptr(s["offsets"]), _ptr(s["lens"]), s["B"], s["T"])
    if kind == "append":
        ld, size, q = s["qkv"].shape[1], s["qkv"].element_size(), s["qkv"].data_ptr()
        _lib.call("aic_hip_kv_append", cache, q, ld, _ptr(s["q"]), H * hd, H, q + H * hd * size, q + (H + Hkv) * hd * size, ld,
                  _ptr(s["cos"]), _ptr(s["sin"]), s["cos"].shape[0], *batch, s["dt"], stream)
        if case["cache"] == "e2m1":
            k, v = s["back"]
            _lib.call("aic_hip_kv_read", cache, _ptr(k), _ptr(v), Hkv * hd, *batch, s["dt"], stream)
        return _appended(s)
    if kind == "bounds":
        _lib.call("aic_hip_kv_bounds", cache, _ptr(s["bounds"]), *batch, stream)
        return s["bounds"]
    if kind == "select":
        _lib.call("aic_hip_kv_select", cache, _ptr(s["bounds"]), _ptr(s["q_in"]), H * hd, *batch, s["max_q"], s["max_len"], H, FIRST, LAST,
                  case["sel"], _ptr(s["picked"]), _ptr(s["picked_lens"]), _ptr(s["ws"]), s["ws"].numel(), s["dt"], stream)
        return s["picked"], s["picked_lens"]
    out = (_ptr(s["q_in"]), H * hd, _ptr(s["o"]), H * hd, _ptr(s["lse"]))
    scale, ws = 1.0 / math.sqrt(hd), (_ptr(s["ws"]), s["ws"].numel(), s["dt"], stream)
    if kind == "attn":
        _lib.call("aic_hip_attn_paged", cache, *out, *batch, s["max_q"], s["max_len"], H, case["window"], scale, *ws)
    else:
        _lib.call("aic_hip_attn_paged_selected", cache, *out, _ptr(s["picked"]), _ptr(s["picked_lens"]), s["T"], case["sel"], H, scale, *ws)
    return (s["o"],) if s["lse"] is None else (s["o"], s["lse"])


# ------------------------------------------------------------------------- the plain forms
def _appended(s):
    """The rotated queries and the cache: its pools, codes as the numbers they are, or its rows as read back."""
    if s["case"]["cache"] == "e2m1":
        return (s["q"],) + s["back"]
    if s["case"]["cache"] == "e4m3":
        return (s["q"],) + tuple(s[k].view(torch.float8_e4m3fn) for k in ("k_pages", "v_pages")) + (s["k_exps"], s["v_exps"])
    return s["q"], s["k_pages"], s["v_pages"]


def _rows(s):
    """Sequence and position of every packed row."""
    t = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["offsets"], t, right=True) - 1
    return b, s["lens"][b] - s["offsets"][b + 1] + t


def _values(s, name, page, slot):
    """fp32 rows [..., Hkv, hd] of the cache at (page, slot)."""
    x = s[name + "_pages"][page, :, slot]
    return x.float() if s[name + "_exps"] is None else _dequantise(x, s[name + "_exps"][page, :, slot], s["case"]["cache"])


def _run_append(s):
    case = s["case"]
    H, Hkv, hd, T = case["H"], case["Hkv"], case["hd"], s["T"]
    b, pos = _rows(s)
    page, slot = s["table"][b, pos // case["ps"]].long(), pos % case["ps"]
    x = s["qkv"].view(T, H + 2 * Hkv, hd).float()
    x1, x2 = x[:, :H + Hkv, :hd // 2], x[:, :H + Hkv, hd // 2:]
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    turned = torch.cat([x1 * c - x2 * sn, x1 * sn + x2 * c], -1)
    s["q"].copy_(turned[:, :H].reshape(T, H * hd))
    for i, (name, y) in enumerate((("k", turned[:, H:]), ("v", x[:, H + Hkv:]))):
        if s[name + "_exps"] is not None:
            y, e = _quantise(y, case["cache"])
            s[name + "_exps"][page, :, slot] = e
        s[name + "_pages"][page, :, slot] = y.to(DT[case["cache"]])
        if case["cache"] == "e2m1":
            s["back"][i].copy_(_values(s, name, page, slot).view(T, Hkv * hd))
    return _appended(s)


def _attend(s, q, at, seen):
    """q [N, R, hd] over the keys at = (page, head, slot), each of them broadcast to [N, L]; seen [N, R, L]."""
    def rows(name):
        x = s[name + "_pages"][at]
        return x.float() if s[name + "_exps"] is None else _dequantise(x, s[name + "_exps"][at], s["case"]["cache"])

    z = torch.matmul(q, rows("k").transpose(1, 2).contiguous()) * (1.0 / math.sqrt(q.shape[-1]))
    z = torch.where(seen, z, -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows("v"))
    return torch.where(total > 0, o / total, torch.zeros_like(o)), (m + torch.log(total)).squeeze(-1)


def _run_attn(s):
    case = s["case"]
    H, Hkv, hd, ps = case["H"], case["Hkv"], case["hd"], case["ps"]
    B, n, L, G = s["B"], s["max_q"], s["max_len"], H // Hkv
    first, lens = s["offsets"][:-1], s["lens"]
    count = s["offsets"][1:] - first
    i = torch.arange(n, device="cuda")
    real = i < count[:, None]                              # [B, n]: rows that exist
    row = (first[:, None] + i).clamp(max=s["T"] - 1)
    j = torch.arange(L, device="cuda")
    page = s["table"][:, (j // ps).clamp(max=s["table"].shape[1] - 1)].long()  # [B, L]
    at = (page.repeat_interleave(Hkv, 0), torch.arange(Hkv, device="cuda").repeat(B)[:, None], (j % ps)[None])
    q = s["q_in"][row].float().view(B, n, Hkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B * Hkv, n * G, hd)
    pos = (lens - count)[:, None] + i                      # [B, n]
    seen = (j <= pos[..., None]) & real[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(B, Hkv, n, G, L).reshape(B * Hkv, n * G, L)
    o, stat = _attend(s, q, at, seen)
    s["o"].copy_(o.view(B, Hkv, n, G, hd).permute(0, 2, 1, 3, 4).reshape(B, n, H * hd)[real])
    if s["lse"] is None:
        return (s["o"],)
    s["lse"].copy_(stat.view(B, Hkv, n, G).permute(0, 2, 1, 3).reshape(B, n, H)[real])
    return s["o"], s["lse"]


def _run_bounds(s):
    case = s["case"]
    ps, Hkv, hd, T = case["ps"], case["Hkv"], case["hd"], s["T"]
    b, pos = _rows(s)
    # the pages that hold the rows: every row's, the same ones several times
    pi = pos // ps
    first = torch.ones(T, dtype=torch.bool, device="cuda")
    first[1:] = (b[1:] != b[:-1]) | (pi[1:] != pi[:-1])
    b, pi = b[first], pi[first]
    page, slot = s["table"][b, pi].long(), torch.arange(ps, device="cuda")
    x = s["k_pages"][page]
    x = x.float() if s["k_exps"] is None else _dequantise(x, s["k_exps"][page], case["cache"])   # [pages, Hkv, ps, hd]
    filled = (slot < (s["lens"][b] - pi * ps)[:, None])[:, None, :, None]
    lo, hi = torch.where(filled, x, math.inf).amin(2), torch.where(filled, x, -math.inf).amax(2)
    s["bounds"][page] = torch.stack([lo, hi], 2).to(s["bounds"].dtype)
    return s["bounds"]


def _pick(s, score, b, pos):
    """The pages of each row and head with the greatest scores, in order of their positions, and the positions they hold."""
    case = s["case"]
    ps, sel = case["ps"], case["sel"]
    count = (pos // ps + 1)[:, None, None]
    at = torch.arange(score.shape[-1], device="cuda")
    score = torch.where((at < FIRST) | (at >= count - LAST), math.inf, score)
    score = torch.where(at < count, score, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :sel]
    if best.shape[-1] < sel:
        best = torch.nn.functional.pad(best, (0, sel - best.shape[-1]), value=score.shape[-1])
    best = torch.sort(torch.where(best < count, best, score.shape[-1]), dim=-1)[0]
    ids = s["table"][b][:, None].expand(-1, best.shape[1], -1).gather(2, best.clamp(max=s["table"].shape[1] - 1))
    picked = torch.where(best < count, ids, -1)
    whole = count[..., 0].clamp(max=sel) - 1
    return picked.to(torch.int32), (whole * ps + (pos % ps)[:, None] + 1).expand(-1, best.shape[1]).contiguous()


def _run_select(s):
    case = s["case"]
    H, Hkv, hd, ps = case["H"], case["Hkv"], case["hd"], case["ps"]
    G, T, P = H // Hkv, s["T"], -(-s["max_len"] // ps)
    b, pos = _rows(s)
    score = torch.empty(T, Hkv, P, dtype=torch.float64, device="cuda")
    first = s["offsets"][:-1]
    count = s["offsets"][1:] - first
    i = torch.arange(s["max_q"], device="cuda")
    real = i < count[:, None]
    row = (first[:, None] + i).clamp(max=T - 1)
    q = s["q_in"][row].double().view(s["B"], s["max_q"], Hkv, G, hd).permute(0, 2, 1, 3, 4).reshape(s["B"] * Hkv, s["max_q"] * G, hd)
    x = s["bounds"][s["table"][:, :P].long()].double().permute(0, 2, 3, 4, 1).reshape(s["B"] * Hkv, 2, hd, P)
    z = torch.matmul(q.clamp(max=0), x[:, 0].contiguous()) + torch.matmul(q.clamp(min=0), x[:, 1].contiguous())
    z = z.view(s["B"], Hkv, s["max_q"], G, P).amax(3).permute(0, 2, 1, 3)
    score.copy_(z[real])
    picked, lens = _pick(s, score, b, pos)
    s["picked"].copy_(picked)
    s["picked_lens"].copy_(lens)
    return s["picked"], s["picked_lens"]


def _run_sparse(s):
    case = s["case"]
    H, Hkv, hd, ps, T = case["H"], case["Hkv"], case["hd"], case["ps"], s["T"]
    G, L = H // Hkv, case["sel"] * ps
    j = torch.arange(L, device="cuda")
    seen = (j < s["picked_lens"].view(-1, 1)).unsqueeze(1).expand(-1, G, -1)
    page = s["picked"].view(T * Hkv, -1).clamp(min=0).long()[:, j // ps]
    at = (page, torch.arange(Hkv, device="cuda").repeat(T)[:, None], (j % ps)[None])
    o, stat = _attend(s, s["q_in"].float().view(T * Hkv, G, hd), at, seen)
    s["o"].copy_(o.view(T, H * hd))
    if s["lse"] is None:
        return (s["o"],)
    s["lse"].copy_(stat.view(T, H))
    return s["o"], s["lse"]


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "attn": _run_attn, "bounds": _run_bounds, "select": _run_select, "sparse": _run_sparse}[
        state["case"]["kind"]](state)


# ------------------------------------------------------------------------------ what it takes
def work(case):
    shape, kind, ps = _shape(case), case["kind"], case["ps"]
    T = sum(n for n, _ in shape)
    H, Hkv, hd, cache = case["H"], case["Hkv"], case["hd"], case["cache"]
    e = 4 if case["dtype"] == "f32" else 2
    side = Hkv * {"f32": 4 * hd, "bf16": 2 * hd, "e4m3": hd + 1, "e2m1": hd // 2 + hd // GROUP}[cache]  # of a cached row: its k or its v
    bound = 2 * Hkv * hd * (4 if cache == "f32" else 2)
    if kind == "append":
        back = T * 2 * (side + Hkv * hd * e) if cache == "e2m1" else 0
        return {"bytes": T * ((2 * H + 2 * Hkv) * hd * e + 2 * side) + max(n for _, n in shape) * hd * 4 + back,
                "flops": T * (6 * (H + Hkv) * hd // 2 + 2 * Hkv * hd)}
    if kind == "bounds":
        pages = [(L - n) // ps for n, L in shape], [(L - 1) // ps for n, L in shape]
        keys = sum(L - lo * ps for (n, L), lo in zip(shape, pages[0]))
        return {"bytes": keys * side + sum(hi - lo + 1 for lo, hi in zip(*pages)) * bound, "flops": 2 * keys * Hkv * hd}
    if kind == "select":
        pages = sum(-(-L // ps) for _, L in shape)
        pairs = sum(sum((L - n + i) // ps + 1 for i in range(n)) for n, L in shape)
        return {"bytes": pages * (bound + 4) + T * (H * hd * e + Hkv * (4 * case["sel"] + 8)), "flops": pairs * H * hd * 4}
    stat = 4 * T * H if case["lse"] else 0
    if kind == "sparse":
        most = case["sel"] * ps
        keys = sum(min(L, n * most) for n, L in shape)
        pairs = sum(sum(min(L - n + i + 1, most) for i in range(n)) for n, L in shape)
        return {"bytes": 2 * T * H * hd * e + 2 * keys * side + T * Hkv * 4 * case["sel"] + stat, "flops": 4 * hd * H * pairs}
    w = case["window"]
    keys = sum(min(L, n + w - 1) if w else L for n, L in shape)
    pairs = sum(sum(min(L - n + i + 1, w or L) for i in range(n)) for n, L in shape)
    return {"bytes": 2 * T * H * hd * e + 2 * keys * side + stat, "flops": 4 * hd * H * pairs}


# ----------------------------------------------------------------------------- in 64 bits
def _two64(e):
    """2^e as float64, exactly, for whole e of any type."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(codes, exps, cache):
    """Codes and biased exponents as float64, from the formats' definitions."""
    if cache == "e2m1":
        c = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
        sign, e, m = 1.0 - 2.0 * (c >> 3), (c >> 1) & 3, (c & 1).double()
        x = torch.where(e > 0, (1 + m / 2) * _two64(e - 1), m / 2)
        return sign * x * _two64(exps.long() - 127).repeat_interleave(GROUP, -1)
    c = codes.long()
    sign, e, m = 1.0 - 2.0 * (c >> 7), (c >> 3) & 15, (c & 7).double()
    x = torch.where(e > 0, (1 + m / 8) * _two64(e - 7), m / 8 * 2.0 ** -6)
    return sign * x * _two64(exps.long() - 127).unsqueeze(-1)


def _round64(x, cache):
    """float64 rows [..., hd] as (the numbers that the cache's codes hold before their powers, the powers' exponents)."""
    top, low, n = (448.0, -6, x.shape[-1]) if cache == "e4m3" else (6.0, 0, GROUP)
    x = x.unflatten(-1, (-1, n))
    most = x.abs().amax(-1)
    e = torch.ceil(torch.log2(most / top))
    e = e + (most > top * _two64(e)).double() - (most <= top * _two64(e - 1)).double()
    y = x * _two64(-e).unsqueeze(-1)
    step = _two64(torch.frexp(y.abs().clamp(min=2.0 ** low))[1] - (4 if cache == "e4m3" else 2))  # the codes' spacing at y
    return torch.round(y / step) * step, e  # to nearest, ties to even


def exact(case, seed):
    s = prepare(case, seed)
    kind, cache, ps = case["kind"], case["cache"], case["ps"]
    ns = (s["offsets"][1:] - s["offsets"][:-1]).tolist()
    offs, lens = s["offsets"].tolist(), s["lens"].tolist()
    H, Hkv, hd = case["H"], case["Hkv"], case["hd"]
    G = H // Hkv
    if kind == "select":
        return None

    def rows(name, page, slot):
        """float64 [len, Hkv, hd]"""
        x = s[name + "_pages"][page, :, slot]
        return x.double() if s[name + "_exps"] is None else _decode64(x, s[name + "_exps"][page, :, slot], cache)

    if kind == "append":
        q = torch.empty(s["T"], H, hd, dtype=torch.float64, device="cuda")
        back = [torch.empty(s["T"], Hkv, hd, dtype=torch.float64, device="cuda") for _ in range(2)]
        pools = [torch.zeros(s["k_pages"].shape, dtype=torch.float64, device="cuda") for _ in range(2)] if cache != "e2m1" else None
        for b, n in enumerate(ns):
            pos = torch.arange(lens[b] - n, lens[b], device="cuda")
            x = s["qkv"][offs[b]:offs[b + 1]].double().view(n, H + 2 * Hkv, hd)
            z = torch.complex(x[..., :hd // 2], x[..., hd // 2:])
            z[:, :H + Hkv] *= torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            y = torch.cat([z.real, z.imag], -1)
            q[offs[b]:offs[b + 1]] = y[:, :H]
            for i in range(2):
                kv = y[:, H + i * Hkv:H + (i + 1) * Hkv]
                if s["k_exps"] is not None:
                    kv, e = _round64(kv, cache)
                    kv = (kv * _two64(e).unsqueeze(-1) if cache == "e2m1" else kv).flatten(-2)
                back[i][offs[b]:offs[b + 1]] = kv
                if pools:
                    pools[i][s["table"][b].long()[pos // ps], :, pos % ps] = kv
        q = q.view(s["T"], H * hd)
        if cache == "e2m1":
            return (q,) + tuple(x.view(s["T"], Hkv * hd) for x in back)
        return (q, *pools) + ((None, None) if cache == "e4m3" else ())
    if kind == "bounds":
        out = torch.zeros(s["bounds"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(ns):
            for pi in range((lens[b] - n) // ps, (lens[b] - 1) // ps + 1):
                page = int(s["table"][b, pi])
                x = rows("k", page, slice(0, lens[b] - pi * ps))
                out[page, :, 0], out[page, :, 1] = x.min(1)[0], x.max(1)[0]
        return out
    outs, stats = [], []
    for b, n in enumerate(ns):
        q = s["q_in"][offs[b]:offs[b + 1]].double().view(n, H, hd) / math.sqrt(hd)
        j = torch.arange(lens[b], device="cuda")
        page = s["table"][b].long()[j // ps]
        full = {name: rows(name, page, j % ps) for name in "kv"}
        at = torch.arange(lens[b] - n, lens[b], device="cuda")[:, None]
        o = torch.empty(n, H, hd, dtype=torch.float64, device="cuda")
        stat = torch.empty(n, H, dtype=torch.float64, device="cuda")
        for h in range(H):
            hide = j > at
            if kind == "attn" and case["window"]:
                hide = hide | (j <= at - case["window"])
            if kind == "sparse":
                # a position is hidden where its page is none of the row's
                chosen = s["picked"][offs[b]:offs[b + 1], h // G]
                held = torch.zeros(n, s["n_pages"] + 1, dtype=torch.bool, device="cuda")
                held.scatter_(1, torch.where(chosen >= 0, chosen.long(), s["n_pages"]), True)
                hide = hide | ~held[:, page]
            z = (q[:, h] @ full["k"][:, h // G].t().contiguous()).masked_fill(hide, -math.inf)
            stat[:, h] = torch.logsumexp(z, -1)
            o[:, h] = torch.exp(z - stat[:, h, None]) @ full["v"][:, h // G].contiguous()
        outs.append(o.view(n, H * hd))
        stats.append(stat)
    return (torch.cat(outs), torch.cat(stats)) if case["lse"] else (torch.cat(outs),)
