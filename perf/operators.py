"""The 8-bit paged key / value cache: appending tokens to it and attending over it.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a serving program holds before the call
    run(state)          one pass: the plain form in torch, or the library's calls where `own`
    work(case)          bytes and operations one pass cannot do without
    exact(case, seed)   the same results in 64 bits

The cache: pages of `page` tokens; page p and KV head h hold E4M3 codes k, v [page, d] and one E8M0
exponent each (value = code 2^(e - 127)). A sequence's position x lies in page table[x // page], slot
x % page. The operators ("op" of a case):
    append   the new tokens' q, k, v rows: bias, rotary embedding, q written out, k and v into the cache
    attend   softmax(q k^T / sqrt(d)) v of the new tokens' query heads over their sequences' positions
             up to their own

A case's sequences: the first has `past` cached tokens and `new` new ones, the others fewer, drawn from
the case alone; the last `idle` of the `b` sequences have no new token. `pad` rows behind the last token
are nobody's and stay as they were.
"""
from __future__ import annotations

import random

import torch

own = False


# ---------------------------------------------------------------- cases

def listed() -> list[dict]:
    qwen = {"h": 14, "kv": 2, "d": 64}    # the 0.5B decoder
    wide = {"h": 32, "kv": 8, "d": 128}   # a 7B-sized decoder with grouped queries
    return [
        # one layer of a chat's next token: latency and launches
        {"name": "append-step-1", "op": "append", "b": 1, "past": 700, "new": 1, "idle": 0, "pad": 0, "page": 16,
         "bias": True, **qwen},
        # 64 conversations decoded together, some of the batch's places empty
        {"name": "append-step-64", "op": "append", "b": 64, "past": 900, "new": 1, "idle": 3, "pad": 3, "page": 32,
         "bias": False, **wide},
        # prompts at once, behind earlier turns, in a row buffer that they do not fill
        {"name": "append-prompts", "op": "append", "b": 4, "past": 777, "new": 1000, "idle": 0, "pad": 50, "page": 64,
         "bias": True, **wide},
        # the attention of the first case
        {"name": "step-700", "op": "attend", "b": 1, "past": 700, "new": 1, "idle": 0, "pad": 0, "page": 16, **qwen},
        # one long document: the cache streams through every compute unit
        {"name": "step-60000", "op": "attend", "b": 1, "past": 60000, "new": 1, "idle": 0, "pad": 0, "page": 64,
         **wide},
        # 64 conversations of very different lengths
        {"name": "step-64", "op": "attend", "b": 64, "past": 4096, "new": 1, "idle": 3, "pad": 3, "page": 32, **wide},
        # 16 query heads on one key head
        {"name": "step-shared-16", "op": "attend", "b": 12, "past": 9000, "new": 1, "idle": 0, "pad": 0, "page": 128,
         "h": 16, "kv": 1, "d": 128},
        # a short question, a whole prompt, a long prompt
        {"name": "prompt-37", "op": "attend", "b": 1, "past": 0, "new": 37, "idle": 0, "pad": 0, "page": 16, **qwen},
        {"name": "prompt-1000", "op": "attend", "b": 1, "past": 0, "new": 1000, "idle": 0, "pad": 24, "page": 32,
         **qwen},
        {"name": "prompt-2048", "op": "attend", "b": 1, "past": 0, "new": 2048, "idle": 0, "pad": 0, "page": 64,
         **wide},
        # a chunk of a document's prompt behind what is cached
        {"name": "chunk-200", "op": "attend", "b": 1, "past": 8000, "new": 200, "idle": 0, "pad": 0, "page": 32,
         **wide},
        # prompts and steps in one call
        {"name": "mixed-24", "op": "attend", "b": 24, "past": 1500, "new": 300, "idle": 1, "pad": 5, "page": 16,
         **qwen},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng) -> dict:
    op = rng.choice(["append", "attend", "attend"])
    kv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "kv": kv, "h": kv * rng.choice([1, 2, 4, 7, 8, 16] if kv < 4 else [1, 2, 4, 7]),
            "d": rng.choice([32, 64, 64, 128, 128]), "page": rng.choice([16, 32, 64, 128])}
    if rng.random() < 0.5:  # steps
        b, past, new = _spread(rng, 1, 64), _spread(rng, 1, 16000), 1
    elif rng.random() < 0.4:  # a prompt or a chunk of one
        b, past, new = 1, rng.choice([0, 0, _spread(rng, 1, 8000)]), _spread(rng, 2, 2048)
    else:  # several prompts, or prompts and steps
        b, past, new = _spread(rng, 2, 24), _spread(rng, 1, 3000), _spread(rng, 2, 700)
    if op == "append":
        past, case["bias"] = min(past, 1200), rng.random() < 0.5
    while b > 1 and (b * case["h"] * new * (past + new) > 2.5e8 or b * (past + new) * kv * case["d"] > 1.4e8):
        b = (b + 1) // 2
    while case["h"] * new * (past + new) > 1.3e8:
        new = new // 2
    return {**case, "b": b, "past": past, "new": new, "idle": rng.randrange(0, 1 + b // 8), "pad": rng.choice([0, 0, 7])}


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Cached and new tokens of each sequence."""
    rng, b, past, new = random.Random(case["b"] * 8191 + case["past"] + 31 * case["new"]), case["b"], case["past"], case["new"]
    pasts = [past] + [int(past * rng.uniform(0.02, 1.0)) for _ in range(b - 1)]
    news = [new] + [1 if rng.random() < 0.5 else rng.randint(1, new) for _ in range(b - 1)]
    return pasts, [0 if i >= b - case["idle"] else n for i, n in enumerate(news)]


# ---------------------------------------------------------------- inputs

def _e8m0(amax: torch.Tensor) -> torch.Tensor:
    """uint8: the smallest exponent with amax <= 448 2^(e - 127)."""
    m, ex = torch.frexp(amax)
    e = (ex - 9 + (m > 0.875) + 127).clamp(0, 254)
    return torch.where(amax > 0, e, torch.zeros_like(e)).to(torch.uint8)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """float32 2^(e - 127) of integers e in 1..254 (0 below)."""
    return (e.to(torch.int32).clamp(min=0) << 23).view(torch.float32)


def _blocks(x: torch.Tensor):
    """(E4M3 codes uint8, E8M0 exponents uint8) of x [pages, kv, page, d]."""
    e = _e8m0(x.abs().amax((2, 3)))
    codes = (x * _pow2(254 - e.int())[:, :, None, None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), e


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, kv, d, page, b = case["h"], case["kv"], case["d"], case["page"], case["b"]
    pasts, news = _lengths(case)
    n = sum(news)
    t = n + case["pad"]
    need = [-(-(p + m) // page) for p, m in zip(pasts, news)]
    pages, wide = sum(need) + 3, max(need) + 1
    # the pool's pages are handed out in no order
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((b, wide), -1, dtype=torch.int32)
    for i, m in enumerate(need):
        table[i, :m] = order[sum(need[:i]):sum(need[:i]) + m]
    starts = torch.tensor([sum(news[:i]) for i in range(b + 1)], dtype=torch.int32)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    gain = torch.where(torch.rand(kv, 1, d, generator=g, device="cuda") < 1 / 16, 6.0, 1.0)  # keys' large channels
    k, ke = _blocks(rnd(pages, kv, page, d) * gain)
    v, ve = _blocks(rnd(pages, kv, page, d) * torch.exp2(2 * rnd(pages, 1, page, 1)))
    s = {"case": case, "n": n, "t": t, "k": k, "ke": ke, "v": v, "ve": ve, "table": table.cuda(),
         "past": torch.tensor(pasts, dtype=torch.int32).cuda(), "q_start": starts.cuda(), "max_new": max(news)}
    if case["op"] == "append":
        qkv = rnd(t, h + 2 * kv, d)
        qkv[:, h:h + kv] *= gain[None, :, 0]
        last = max(p + m for p, m in zip(pasts, news))
        inv = 1.0 / 1e6 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        ang = torch.arange(last, device="cuda", dtype=torch.float64)[:, None] * inv
        return {**s, "qkv": qkv.reshape(t, -1), "bias": rnd((h + 2 * kv) * d) * 0.3 if case["bias"] else None,
                "cos": ang.cos().float(), "sin": ang.sin().float(), "out": rnd(t, h * d)}
    return {**s, "q": rnd(t, h * d) * 1.5, "out": rnd(t, h * d)}


# ---------------------------------------------------------------- the plain form

def _rows(s: dict):
    """Sequence and place in it of each new token."""
    rows = torch.arange(s["n"], device="cuda", dtype=torch.int32)
    seq = torch.bucketize(rows, s["q_start"][1:], right=True)
    return seq, rows - s["q_start"][seq]


def _put(codes, e, y, pg, slot):
    """y [n, kv, d] into slots `slot` of pages `pg`: the blocks' exponents grow where a new token needs it."""
    pages, kv, page, _ = codes.shape
    big = torch.zeros(pages, kv, device="cuda").scatter_reduce_(0, pg[:, None].expand(-1, kv), y.abs().amax(2), "amax")
    first = torch.full((pages,), page, device="cuda").scatter_reduce_(0, pg, slot, "amin")
    e_old = torch.where((first == 0)[:, None], torch.zeros_like(e), e)
    e_new = torch.where((first < page)[:, None], torch.maximum(e_old, _e8m0(big)), e)
    shift = _pow2(127 + e_old.int() - e_new.int())[:, :, None, None]
    moved = (codes.view(torch.float8_e4m3fn).float() * shift).to(torch.float8_e4m3fn).view(torch.uint8)
    old = (torch.arange(page, device="cuda") < first[:, None]) & (first < page)[:, None]
    codes.copy_(torch.where(old[:, None, :, None], moved, codes))
    codes[pg, :, slot] = (y * _pow2(254 - e_new.int())[pg][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    e.copy_(e_new)


def _plain_append(s: dict):
    c, n = s["case"], s["n"]
    h, kv, d, page = c["h"], c["kv"], c["d"], c["page"]
    seq, i = _rows(s)
    pos = s["past"][seq] + i
    x = s["qkv"][:n]
    x = (x if s["bias"] is None else x + s["bias"]).reshape(n, h + 2 * kv, d)
    a, b = x[:, :h + kv, :d // 2], x[:, :h + kv, d // 2:]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    s["out"][:n] = y[:, :h].reshape(n, -1)
    pg, slot = s["table"][seq, pos // page].long(), (pos % page).long()
    _put(s["k"], s["ke"], y[:, h:].contiguous(), pg, slot)
    _put(s["v"], s["ve"], x[:, h + kv:].contiguous(), pg, slot)


def _held(codes, e, table):
    """float32 [b, kv, positions, d] of what the tables' pages hold."""
    at = table.clamp(min=0).long()
    x = codes[at].view(torch.float8_e4m3fn).float() * _pow2(e[at])[:, :, :, None, None]
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _plain_attend(s: dict):
    c = s["case"]
    h, kv, d, new, b = c["h"], c["kv"], c["d"], s["max_new"], c["b"]
    at = (s["q_start"][:-1, None] + torch.arange(new, device="cuda")).clamp(max=s["t"] - 1)
    q = s["q"][at].reshape(b, new, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)
    k, v = _held(s["k"], s["ke"], s["table"]), _held(s["v"], s["ve"], s["table"])
    sc = q @ k.transpose(2, 3) / d ** 0.5
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= (s["past"][:, None] + torch.arange(new, device="cuda"))[:, :, None]) \
        & (s["table"] >= 0).repeat_interleave(c["page"], 1)[:, None]
    sc = sc.reshape(b, kv, new, -1, k.shape[2]).masked_fill(~seen[:, None, :, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    o = (p.reshape(b, kv, -1, k.shape[2]) @ v).reshape(p.shape[:-1] + (d,)) / torch.where(l > 0, l, torch.ones_like(l))
    seq, i = _rows(s)
    s["out"][:s["n"]] = o.permute(0, 2, 1, 3, 4).reshape(b, new, h * d)[seq, i]


# ---------------------------------------------------------------- the library's calls

def _handle(s: dict):
    """The argument structures and the workspace that a program keeps between calls."""
    import ctypes as C

    from lowbit_amd import kernels as K
    c, p, L = s["case"], (lambda t: None if t is None else t.data_ptr()), K.lib()
    pool = K.LbdKv8Pool(p(s["k"]), p(s["v"]), p(s["ke"]), p(s["ve"]), s["k"].shape[0], c["page"], c["kv"], c["d"])
    batch = K.LbdKv8Batch(p(s["q_start"]), p(s["past"]), p(s["table"]), c["b"], s["table"].shape[1], s["max_new"],
                          s["t"])
    stream, args = torch.cuda.current_stream().cuda_stream, (C.byref(pool), C.byref(batch))
    if c["op"] == "append":
        width = s["qkv"].shape[1]
        call = (L.lbd_kv8_append, (*args, p(s["qkv"]), width, p(s["bias"]), c["h"], p(s["cos"]), p(s["sin"]),
                                   s["cos"].shape[0], p(s["out"]), c["h"] * c["d"], stream))
        return call, (K._check, pool, batch)
    need = L.lbd_kv8_attention_work_bytes(*args, c["h"])
    ws = torch.empty(max(256, need), dtype=torch.uint8, device="cuda")
    call = (L.lbd_kv8_attention, (*args, p(s["q"]), c["h"] * c["d"], c["h"], p(s["out"]), c["h"] * c["d"], p(ws), need,
                                  stream))
    return call, (K._check, pool, batch, ws)


def run(s: dict):
    if own:
        if "handle" not in s:
            s["handle"] = _handle(s)
        (fn, args), keep = s["handle"]
        keep[0](fn(*args), "kv8", False)
    elif s["case"]["op"] == "append":
        _plain_append(s)
    else:
        _plain_attend(s)
    if s["case"]["op"] == "attend":
        return s["out"]
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return {"q": s["out"], "k": s["k"].view(e4m3), "v": s["v"].view(e4m3), "ke": s["ke"].view(e8m0),
            "ve": s["ve"].view(e8m0)}


# ---------------------------------------------------------------- work

def work(case: dict) -> dict:
    h, kv, d, (pasts, news) = case["h"], case["kv"], case["d"], _lengths(case)
    n = sum(news)
    if case["op"] == "append":
        blocks = sum(-(-(p + m) // case["page"]) - p // case["page"] for p, m in zip(pasts, news) if m)
        return {"bytes": n * (4 * (h + 2 * kv) * d + 4 * d + 4 * h * d + 2 * kv * d) + 2 * kv * blocks,
                "flops": n * 3 * (h + 2 * kv) * d}
    keys = sum(p + m for p, m in zip(pasts, news) if m)
    pairs = sum(m * p + m * (m + 1) / 2 for p, m in zip(pasts, news))
    return {"bytes": 8 * n * h * d + 2 * kv * keys * (d + 1 / case["page"]), "flops": 4 * pairs * h * d}


# ---------------------------------------------------------------- the results in 64 bits

def _values(codes: torch.Tensor) -> torch.Tensor:
    """float64 that E4M3 bytes stand for."""
    c = codes.long()
    ex, man = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(ex > 0, (8 + man) * torch.pow(2.0, ex.double() - 10), man * 2.0 ** -9)
    return torch.where(c > 127, -mag, mag)


def _nearest(x: torch.Tensor) -> torch.Tensor:
    """float64 x, at most 448 in magnitude, on the E4M3 grid."""
    step = torch.pow(2.0, torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(s: dict):
    c = s["case"]
    h, kv, d, page = c["h"], c["kv"], c["d"], c["page"]
    pasts, news = _lengths(c)
    out, k, v = s["out"].double(), _values(s["k"]), _values(s["v"])
    ke, ve, row, table = s["ke"].double(), s["ve"].double(), 0, s["table"].tolist()
    for b, (past, new) in enumerate(zip(pasts, news)):
        if not new:
            continue
        x = s["qkv"][row:row + new].double() + (0 if s["bias"] is None else s["bias"].double())
        x = x.reshape(new, h + 2 * kv, d)
        cos, sin = (s[t][past:past + new].double()[:, None] for t in ("cos", "sin"))
        a, z = x[:, :h + kv].split(d // 2, 2)
        y = torch.cat([a * cos - z * sin, z * cos + a * sin], 2)
        out[row:row + new] = y[:, :h].reshape(new, -1)
        at = past
        while at < past + new:
            end = min(past + new, (at // page + 1) * page)
            pg, lo, hi = table[b][at // page], at % page, at % page + end - at
            for codes, ex, new_rows in ((k, ke, y[:, h:]), (v, ve, x[:, h + kv:])):
                t = new_rows[at - past:end - past].transpose(0, 1)
                want = torch.ceil(torch.log2(t.abs().amax((1, 2)) / 448)).clamp(min=-127) + 127
                was = ex[pg] if lo else torch.zeros_like(want)
                now = torch.maximum(was, want)
                codes[pg, :, :lo] = _nearest(codes[pg, :, :lo] * torch.pow(2.0, was - now)[:, None, None])
                codes[pg, :, lo:hi] = _nearest(t * torch.pow(2.0, 127 - now)[:, None, None])
                ex[pg] = now
            at = end
        row += new
    return {"q": out, "k": k, "v": v, "ke": torch.pow(2.0, ke - 127), "ve": torch.pow(2.0, ve - 127)}


def _exact_attend(s: dict):
    c = s["case"]
    h, kv, d = c["h"], c["kv"], c["d"]
    out, row, (pasts, news) = s["out"].double(), 0, _lengths(c)
    for b, (past, new) in enumerate(zip(pasts, news)):
        if not new:
            continue
        pages = s["table"][b, :-(-(past + new) // c["page"])].long()
        flat = lambda codes, e: (_values(codes[pages]) * torch.pow(2.0, e[pages].double() - 127)[:, :, None, None]  # noqa: E731
                                 ).transpose(0, 1).reshape(kv, -1, d)[:, :past + new]
        k, v = flat(s["k"], s["ke"]), flat(s["v"], s["ve"])
        hidden = torch.arange(past + new, device="cuda") > past + torch.arange(new, device="cuda")[:, None]
        for j in range(h):
            q = s["q"][row:row + new, j * d:(j + 1) * d].double()
            sc = (q @ k[j // (h // kv)].t() / d ** 0.5).masked_fill(hidden, float("-inf"))
            out[row:row + new, j * d:(j + 1) * d] = torch.softmax(sc, 1) @ v[j // (h // kv)]
        row += new
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)
