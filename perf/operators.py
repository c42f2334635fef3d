"""What the operators of serving over a paged key/value cache are measured on.

One pass writes a ragged batch's new keys and values into the cache, reads cached rows back, attends
from the new tokens over the cache, or verifies drafted tokens against the target's logits.  `run`
computes each in plain torch operations, or calls the library where `own` is true.  Sizes follow the
model widths that the library is benchmarked on (12 heads of 64, 16 heads of 128, 4 heads of 32;
vocabulary 32000) and grouped key/value heads of them.

A batch is `B` sequences; sequence b brings the rows offsets[b] .. offsets[b + 1] of the packed
inputs and its cache holds lens[b] tokens with them.  Lengths come from the case alone (_shape), the
order of the sequences, the pages' places and all values from the seed.
"""
import ctypes
import math

import torch

own = False

V_MAIN = 32000  # the benchmark models' vocabulary
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.uint8}
E4M3_MAX = 448.0


def listed():
    return [
        # one token of each of four chat sequences, written as it is: the smallest call of a decode step
        dict(name="write_decode_125m", kind="write", B=4, n=1, L=700, H=12, Hkv=12, hd=64, ps=16, cache="bf16", dtype="bf16"),
        # prompts of up to 2048 tokens at the 1B width with eight key/value heads, quantised as they are written
        dict(name="write_prompt_e4m3", kind="write", B=8, n=2048, L=2048, H=16, Hkv=8, hd=128, ps=64, cache="e4m3", dtype="bf16"),
        # one sequence's cache read back to be moved or looked at
        dict(name="read_one_e4m3", kind="read", B=1, n=777, L=777, H=16, Hkv=4, hd=128, ps=16, cache="e4m3", dtype="bf16"),
        # all caches of a batch read back at the 1B width
        dict(name="read_batch_e4m3", kind="read", B=16, n=4096, L=4096, H=16, Hkv=8, hd=128, ps=64, cache="e4m3", dtype="bf16"),
        # single-token decoding of one chat sequence at the 125M widths: latency
        dict(name="decode_125m_b1", kind="attn", B=1, n=1, L=513, H=12, Hkv=12, hd=64, ps=16, window=0, cache="bf16",
             dtype="bf16", lse=False),
        # single-token decoding of a ragged batch of long contexts, grouped heads, quantised cache
        dict(name="decode_e4m3_b32", kind="attn", B=32, n=1, L=8000, H=16, Hkv=2, hd=128, ps=64, window=0, cache="e4m3",
             dtype="bf16", lse=False),
        # the largest decode: 16-bit cache of eight key/value heads, contexts up to 16384
        dict(name="decode_bf16_b32", kind="attn", B=32, n=1, L=16384, H=16, Hkv=8, hd=128, ps=64, window=0, cache="bf16",
             dtype="bf16", lse=False),
        # the target's pass over up to four drafted tokens and the one before them, for 16 sequences
        dict(name="verify_pass_b16", kind="attn", B=16, n=5, L=3000, H=16, Hkv=16, hd=128, ps=16, window=0, cache="e4m3",
             dtype="bf16", lse=False),
        # a 2048-token chunk of one long prompt behind 6144 cached tokens
        dict(name="chunk_2048_of_8192", kind="attn", B=1, n=2048, L=8192, H=16, Hkv=2, hd=128, ps=64, window=0, cache="bf16",
             dtype="bf16", lse=False),
        # fp32 parity configuration: short prompts of the tiny model in one ragged batch, with row statistics
        dict(name="tiny_f32_prompts", kind="attn", B=8, n=200, L=333, H=4, Hkv=4, hd=32, ps=24, window=100, cache="f32",
             dtype="f32", lse=True),
        # four drafted tokens of one sequence against the target: latency
        dict(name="drafts_b1", kind="drafts", B=1, n=5, V=V_MAIN, temperature=0.8, draft="logits", dtype="f32"),
        # up to seven drafted tokens for each of 64 sequences
        dict(name="drafts_b64", kind="drafts", B=64, n=8, V=V_MAIN, temperature=1.0, draft="logits", dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "attn", "attn", "drafts"])
    if kind == "drafts":
        n = rng.randint(1, 8)
        return dict(kind=kind, B=_log(rng, 1, 64), n=n, V=rng.choice([512, V_MAIN, V_MAIN, _log(rng, 100, V_MAIN)]),
                    temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), draft=rng.choice(["logits", "logits", "none"]),
                    dtype=rng.choice(["f32", "f32", "bf16"]))
    H, hd = rng.choice([(12, 64), (16, 64), (16, 128), (16, 128), (4, 32)])
    G = rng.choice([1, 2, 4] if H < 16 else [1, 2, 8] if hd == 128 else [2, 4, 8])
    cache = rng.choice(["bf16", "bf16", "e4m3", "e4m3", "f32"])
    dtype = "f32" if cache == "f32" else "bf16"
    case = dict(kind=kind, H=H, Hkv=H // G, hd=hd, ps=rng.choice([16, 16, 24, 32, 64, 64, 128]), cache=cache, dtype=dtype)
    if kind in ("write", "read"):
        B = _log(rng, 1, 32)
        n = rng.choice([1, _log(rng, 1, 4096 // B)]) if kind == "write" else _log(rng, 1, 16384 // B)
        return dict(case, B=B, n=n, L=n + rng.choice([0, _log(rng, 1, 1000)]) if kind == "write" else n)
    # tokens that come in together: one, a few drafted ones, a chunk of a prompt
    few = 1 if rng.random() < 0.4 else rng.randint(2, 8)
    n = few if rng.random() < 0.6 else _log(rng, 9, 1024)
    B = _log(rng, 1, 30) if n <= 8 else _log(rng, 1, max(1, min(16, 2048 // n)))
    top = 8000 if n <= 8 and dtype != "f32" else 4096 if dtype != "f32" else 1024
    return dict(case, B=B, n=n, L=n + _log(rng, 1, top), window=rng.choice([0, 0, 0, _log(rng, 16, 2000)]),
                lse=rng.random() < 0.3)


# ----------------------------------------------------------------------------------- inputs
def _shape(case):
    """(n_b, len_b) of each sequence, longest first: sequence 0 has the case's n and L, the others
    down to a quarter of them, spread evenly."""
    got = []
    for b in range(case["B"]):
        f = 1.0 if b == 0 else 0.25 + 0.75 * ((b * 0.6180339887498949) % 1.0)
        n = max(1, round(case["n"] * f))
        got.append((n, n if case["kind"] == "drafts" else max(n, round(case["L"] * f)) if case["kind"] == "attn" or case["L"] > case["n"] else n))
    return got


def _heads(case):
    return case["H"], case["Hkv"], case["hd"]


def _scale_bits(amax):
    """Power-of-two exponent e of each amax: the least with amax <= 448 * 2^e, at least -126."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e.clamp(min=-126), torch.zeros_like(e))


def _pow2(e):
    """2^e in fp32, exactly, for whole e in -126 .. 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """fp32 [..., hd] -> (e4m3 codes as bytes, biased exponents [...])."""
    e = _scale_bits(x.abs().amax(-1))
    codes = (x * _pow2(-e).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    shape = _shape(case)
    order = torch.randperm(len(shape), generator=g, device="cuda").tolist()
    shape = [shape[i] for i in order]
    ns = [n for n, _ in shape]
    T, B = sum(ns), len(ns)
    offsets = torch.tensor([sum(ns[:b]) for b in range(B + 1)], device="cuda")
    s = dict(case=case, B=B, T=T, max_q=max(ns), max_len=max(n for _, n in shape), offsets=offsets)
    if case["kind"] == "drafts":
        V, t = case["V"], DT[case["dtype"]]
        # peaked logits, as a language model's; the draft model's are near them
        z = randn(T, V) * 2.5
        d = z + randn(T, V) * 0.7
        s.update(logits=z.to(t), draft=d.to(t) if case["draft"] == "logits" else None)
        # the draft's own choices, row t's for token t + 1
        temp = max(case["temperature"], 1e-2)
        picks = torch.multinomial(torch.softmax(d.to(t).float() / temp, -1), 1, generator=g)[:, 0]
        s["ids"] = torch.cat([torch.randint(0, V, (1,), generator=g, device="cuda"), picks[:-1]])
        s["u"], s["u_next"] = torch.rand(T, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
        s["lens"] = torch.tensor([100 + n for n in ns], device="cuda") + torch.randint(0, 1000, (B,), generator=g, device="cuda")
        s["out"] = (torch.empty(B, s["max_q"], dtype=torch.int64, device="cuda"),
                    torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int64, device="cuda"))
        if own:
            _drafts_workspace(s)
        return s
    H, Hkv, hd = _heads(case)
    t, ps = DT[case["dtype"]], case["ps"]
    lens = [n for _, n in shape]
    pages = [-(-n // ps) for n in lens]
    width, n_pages = max(pages) + 1, sum(pages) + 3
    places = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    for b in range(B):
        at = sum(pages[:b])
        table[b, :pages[b]] = places[at:at + pages[b]]
    s.update(lens=torch.tensor(lens, device="cuda"), table=table, n_pages=n_pages)
    pool = (n_pages, Hkv, ps, hd)
    if case["kind"] == "write":
        # the pool before the call, and the rows of a fused q/k/v projection
        s["k_pages"], s["v_pages"] = (torch.zeros(pool, dtype=DT[case["cache"]], device="cuda") for _ in range(2))
        s["k_exps"], s["v_exps"] = (torch.zeros(pool[:3], dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        channel = 1.0 + 3.0 * (torch.rand(Hkv, 1, hd, generator=g, device="cuda") > 0.95)  # keys have a few loud channels
        for name, x in (("k", randn(*pool) * channel), ("v", randn(*pool))):
            if case["cache"] == "e4m3":
                s[name + "_pages"], s[name + "_exps"] = _quantise(x)
            else:
                s[name + "_pages"], s[name + "_exps"] = x.to(DT[case["cache"]]), None
    if case["kind"] == "read":
        s["out"] = tuple(torch.empty(T, Hkv * hd, dtype=t, device="cuda") for _ in range(2))
    else:
        s["qkv"] = randn(T, (H + 2 * Hkv) * hd).to(t)
    if case["kind"] == "attn":
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
    code = {"f32": _lib.AIC_F32, "bf16": _lib.AIC_BF16, "e4m3": _lib.AIC_U8}
    e4m3 = case["cache"] == "e4m3"
    s["cache"] = _lib.KVPages(_ptr(s["k_pages"]), _ptr(s["v_pages"]), _ptr(s["k_exps"]) if e4m3 else None,
                              _ptr(s["v_exps"]) if e4m3 else None, _ptr(s["table"]), s["table"].shape[1], s["n_pages"],
                              case["ps"], case["Hkv"], case["hd"], code[case["cache"]])
    s["dt"] = code[case["dtype"]]
    if case["kind"] == "attn":
        n = _lib.load().aic_hip_attn_paged_workspace(ctypes.byref(s["cache"]), s["B"], s["T"], s["max_q"], s["max_len"], case["H"])
        s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")


def _drafts_workspace(s):
    from autonomousaicore_amd import _lib
    s["dt"] = _lib.AIC_F32 if s["case"]["dtype"] == "f32" else _lib.AIC_BF16
    n = _lib.load().aic_hip_verify_drafts_workspace(s["B"], s["T"], s["case"]["V"])
    s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")


def _run_own(s):
    from autonomousaicore_amd import _lib
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    batch = (_ptr(s["offsets"]), _ptr(s["lens"]), s["B"], s["T"])
    if case["kind"] == "drafts":
        V = case["V"]
        tokens, counts, lens = s["out"]
        _lib.call("aic_hip_verify_drafts", _ptr(s["logits"]), V, _ptr(s["draft"]), V, _ptr(s["ids"]), _ptr(s["u"]),
                  _ptr(s["u_next"]), *batch, s["max_q"], V, case["temperature"], _ptr(tokens), _ptr(counts), _ptr(lens),
                  _ptr(s["ws"]), s["ws"].numel(), s["dt"], stream)
        return s["out"]
    H, Hkv, hd = _heads(case)
    cache = ctypes.byref(s["cache"])
    if case["kind"] == "read":
        k, v = s["out"]
        _lib.call("aic_hip_kv_read", cache, _ptr(k), _ptr(v), Hkv * hd, *batch, s["dt"], stream)
        return s["out"]
    ld, size, q = s["qkv"].shape[1], s["qkv"].element_size(), s["qkv"].data_ptr()
    if case["kind"] == "write":
        _lib.call("aic_hip_kv_write", cache, q + H * hd * size, q + (H + Hkv) * hd * size, ld, *batch, s["dt"], stream)
        return _written(s)
    _lib.call("aic_hip_attn_paged", cache, q, ld, _ptr(s["o"]), H * hd, _ptr(s["lse"]), *batch, s["max_q"], s["max_len"], H,
              case["window"], 1.0 / math.sqrt(hd), _ptr(s["ws"]), s["ws"].numel(), s["dt"], stream)
    return (s["o"],) if s["lse"] is None else (s["o"], s["lse"])


# ------------------------------------------------------------------------- the plain forms
def _written(s):
    """The cache's two pools; codes as the e4m3 numbers they are, with their exponents."""
    if s["case"]["cache"] != "e4m3":
        return s["k_pages"], s["v_pages"]
    return tuple(s[k].view(torch.float8_e4m3fn) for k in ("k_pages", "v_pages")) + (s["k_exps"], s["v_exps"])


def _places(s):
    """(page, slot) of every packed row."""
    t = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["offsets"], t, right=True) - 1
    pos = s["lens"][b] - s["offsets"][b + 1] + t
    ps = s["case"]["ps"]
    return s["table"][b, pos // ps].long(), pos % ps


def _values(s, name, page, slot):
    """fp32 rows [..., Hkv, hd] of the cache at (page, slot)."""
    x = s[name + "_pages"][page, :, slot]
    if s["case"]["cache"] != "e4m3":
        return x.float()
    return x.view(torch.float8_e4m3fn).float() * _pow2(s[name + "_exps"][page, :, slot].int() - 127).unsqueeze(-1)


def _run_write(s):
    H, Hkv, hd = _heads(s["case"])
    page, slot = _places(s)
    rows = s["qkv"][:, H * hd:].view(s["T"], 2, Hkv, hd)
    for i, name in enumerate("kv"):
        x = rows[:, i]
        if s["case"]["cache"] == "e4m3":
            x, e = _quantise(x.float())
            s[name + "_exps"][page, :, slot] = e
        s[name + "_pages"][page, :, slot] = x
    return _written(s)


def _run_read(s):
    page, slot = _places(s)
    for name, out in zip("kv", s["out"]):
        out.copy_(_values(s, name, page, slot).view(out.shape))
    return s["out"]


def _run_attn(s):
    case = s["case"]
    H, Hkv, hd = _heads(case)
    B, n, L, G, ps = s["B"], s["max_q"], s["max_len"], H // Hkv, case["ps"]
    first, lens = s["offsets"][:-1], s["lens"]
    count = s["offsets"][1:] - first
    i = torch.arange(n, device="cuda")
    real = i < count[:, None]                              # [B, n]: rows that exist
    row = (first[:, None] + i).clamp(max=s["T"] - 1)
    j = torch.arange(L, device="cuda")
    page = s["table"][:, (j // ps).clamp(max=s["table"].shape[1] - 1)].long()  # [B, L]
    slot = (j % ps).expand(B, L)

    def heads(name):                                       # [B * Hkv, L, hd]
        return _values(s, name, page, slot).permute(0, 2, 1, 3).reshape(B * Hkv, L, hd)

    q = s["qkv"][row][..., :H * hd].float().view(B, n, Hkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B * Hkv, n * G, hd)
    z = torch.matmul(q, heads("k").transpose(1, 2).contiguous()).view(B, Hkv, n, G, L) * (1.0 / math.sqrt(hd))
    pos = (lens - count)[:, None] + i                      # [B, n]
    seen = (j <= pos[..., None]) & real[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    z = torch.where(seen[:, None, :, None], z, -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B * Hkv, n * G, L), heads("v")).view(B, Hkv, n, G, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(B, n, H * hd)
    s["o"].copy_(o[real])
    if s["lse"] is None:
        return (s["o"],)
    s["lse"].copy_((m + torch.log(total)).squeeze(-1).permute(0, 2, 1, 3).reshape(B, n, H)[real])
    return s["o"], s["lse"]


def _run_drafts(s):
    case = s["case"]
    B, n, T, V = s["B"], s["max_q"], s["T"], case["V"]
    first = s["offsets"][:-1]
    count = s["offsets"][1:] - first
    i = torch.arange(n, device="cuda")
    row = (first[:, None] + i).clamp(max=T - 1)
    x = s["ids"][(row + 1).clamp(max=T - 1)]               # the draft that row (b, i) judges
    judged = i < count[:, None] - 1
    z = s["logits"].double()
    if case["temperature"] <= 0.001:
        best = z.argmax(-1)[row]
        kept = ((best == x) & judged).long().cumprod(1).sum(1)
        new = best.gather(1, kept[:, None])[:, 0]
    else:
        p = torch.softmax(z / case["temperature"], -1)
        if s["draft"] is None:
            px, dx = p[row, x], torch.ones_like(x, dtype=torch.float64)
        else:
            d = torch.softmax(s["draft"].double() / case["temperature"], -1)
            px, dx = p[row, x], d[row, x]
        kept = ((s["u"][row].double() * dx < px) & judged).long().cumprod(1).sum(1)
        at = row.gather(1, kept[:, None])[:, 0]
        mass, short = p[at], kept < count - 1
        if s["draft"] is None:
            off = torch.zeros_like(mass).scatter_(1, x.gather(1, kept[:, None]), 1.0)
        else:
            off = d[at]
        left = torch.where(short[:, None], (mass - off).clamp(min=0), mass)
        cdf = left.cumsum(-1)
        new = torch.searchsorted(cdf, cdf[:, -1:] * s["u_next"].double()[:, None], right=True)[:, 0].clamp(max=V - 1)
    tokens, counts, lens = s["out"]
    tokens.copy_(torch.where(i < kept[:, None], x, torch.where(i == kept[:, None], new[:, None], -1)))
    counts.copy_(kept + 1)
    lens.copy_(s["lens"] - count + kept + 1)
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"write": _run_write, "read": _run_read, "attn": _run_attn, "drafts": _run_drafts}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------ what it takes
def work(case):
    shape = _shape(case)
    T = sum(n for n, _ in shape)
    if case["kind"] == "drafts":
        e = 4 if case["dtype"] == "f32" else 2
        rows = T + (T - case["B"] if case["draft"] == "logits" and case["temperature"] > 0.001 else 0)
        return {"bytes": rows * case["V"] * e + T * 20 + case["B"] * 40, "flops": rows * case["V"] * 4}
    H, Hkv, hd = _heads(case)
    e = 4 if case["dtype"] == "f32" else 2
    row = 2 * Hkv * (hd + 1 if case["cache"] == "e4m3" else hd * (4 if case["cache"] == "f32" else 2))  # of the cache
    if case["kind"] != "attn":
        return {"bytes": T * (2 * Hkv * hd * e + row), "flops": T * 2 * Hkv * hd}
    w = case["window"]
    keys = sum(min(L, n + w - 1) if w else L for n, L in shape)
    pairs = sum(sum(min(L - n + i + 1, w or L) for i in range(n)) for n, L in shape)
    return {"bytes": 2 * T * H * hd * e + keys * row + (4 * T * H if case["lse"] else 0), "flops": 4 * hd * H * pairs}


# ----------------------------------------------------------------------------- in 64 bits
def _two64(e):
    """2^e as float64, exactly, for whole e of any type."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(codes, exps):
    """e4m3 codes and biased exponents as float64, from the format's definition."""
    c = codes.long()
    sign, e, m = 1.0 - 2.0 * (c >> 7), (c >> 3) & 15, (c & 7).double()
    x = torch.where(e > 0, (1 + m / 8) * _two64(e - 7), m / 8 * 2.0 ** -6)
    return sign * x * _two64(exps.long() - 127).unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    ns = (s["offsets"][1:] - s["offsets"][:-1]).tolist()
    offs, lens = s["offsets"].tolist(), s["lens"].tolist()
    if case["kind"] == "drafts":
        return _exact_drafts(s, case, offs, ns, lens)
    H, Hkv, hd = _heads(case)
    ps = case["ps"]

    def slots(b, pos):
        return s["table"][b].long()[pos // ps], pos % ps

    if case["kind"] == "write":
        names = ("k_pages", "v_pages", "k_exps", "v_exps") if case["cache"] == "e4m3" else ("k_pages", "v_pages")
        out = [torch.zeros(s[k].shape, dtype=torch.float64 if "pages" in k else torch.int64, device="cuda") for k in names]
        for b, n in enumerate(ns):
            page, slot = slots(b, torch.arange(lens[b] - n, lens[b], device="cuda"))
            for i in range(2):
                x = s["qkv"][offs[b]:offs[b + 1], (H + i * Hkv) * hd:(H + (i + 1) * Hkv) * hd].double().view(n, Hkv, hd)
                if case["cache"] == "e4m3":
                    top = x.abs().amax(-1)
                    e = torch.ceil(torch.log2(top / E4M3_MAX))
                    e = e + (top > E4M3_MAX * _two64(e)).double() - (top <= E4M3_MAX * _two64(e - 1)).double()
                    out[2 + i][page, :, slot] = e.long() + 127
                    y = x * _two64(-e).unsqueeze(-1)
                    step = _two64(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)  # e4m3's spacing at y
                    x = torch.round(y / step) * step  # to nearest, ties to even
                out[i][page, :, slot] = x
        return tuple(out)
    full = {}
    for name in "kv":
        full[name] = [None] * len(ns)
        for b in range(len(ns)):
            page, slot = slots(b, torch.arange(lens[b], device="cuda"))
            x = s[name + "_pages"][page, :, slot]
            full[name][b] = _decode64(x, s[name + "_exps"][page, :, slot]) if case["cache"] == "e4m3" else x.double()
    if case["kind"] == "read":
        return tuple(torch.cat([full[k][b][lens[b] - n:].reshape(n, -1) for b, n in enumerate(ns)]) for k in "kv")
    outs, stats = [], []
    for b, n in enumerate(ns):
        q = s["qkv"][offs[b]:offs[b + 1], :H * hd].double().view(n, H, hd)
        at = torch.arange(lens[b] - n, lens[b], device="cuda")[:, None]
        j = torch.arange(lens[b], device="cuda")
        hide = (j > at) | ((j <= at - case["window"]) if case["window"] else False)
        heads = []
        for h in range(H):
            z = (q[:, h] @ full["k"][b][:, h * Hkv // H].t().contiguous()) / math.sqrt(hd)
            z = z.masked_fill(hide, -math.inf)
            stat = torch.logsumexp(z, -1)
            heads.append((torch.exp(z - stat[:, None]) @ full["v"][b][:, h * Hkv // H].contiguous(), stat))
        outs.append(torch.stack([o for o, _ in heads], 1).view(n, H * hd))
        stats.append(torch.stack([t for _, t in heads], 1))
    return (torch.cat(outs), torch.cat(stats)) if case["lse"] else (torch.cat(outs),)


def _exact_drafts(s, case, offs, ns, lens):
    B, T = s["B"], case["temperature"]
    tokens = torch.full((B, s["max_q"]), -1)
    counts, out_lens = [], []
    ids, u, u_next = s["ids"].tolist(), s["u"].double().tolist(), s["u_next"].double().tolist()

    def dist(row):
        z = row.double() / T
        w = torch.exp(z - z.max())
        return w / w.sum()

    for b, n in enumerate(ns):
        got, nxt = [], None
        for i in range(n):
            t = offs[b] + i
            if T <= 0.001:
                p = torch.zeros(case["V"], dtype=torch.float64, device="cuda")
                p[int(s["logits"][t].double().argmax())] = 1.0
            else:
                p = dist(s["logits"][t])
            if i == n - 1:
                nxt = p
                break
            x = ids[t + 1]
            if T <= 0.001 or s["draft"] is None:
                d = torch.zeros_like(p)
                d[x] = 1.0
            else:
                d = dist(s["draft"][t])
            if u[t] * float(d[x]) < float(p[x]):
                got.append(x)
            else:
                nxt = torch.relu(p - d)
                break
        c = torch.cumsum(nxt, 0)
        got.append(int((c <= c[-1] * u_next[b]).sum().clamp(max=case["V"] - 1)))
        tokens[b, :len(got)] = torch.tensor(got)
        counts.append(len(got))
        out_lens.append(lens[b] - n + len(got))
    return tokens, torch.tensor(counts), torch.tensor(out_lens)
