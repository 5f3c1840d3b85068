"""The paged 8-bit cache under windows and beams: attention with a sliding window and sinks, copies of
pages, beam search's selection, and the beams' states put in their new order.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a serving program holds before the call
    run(state)          one pass: the plain form in torch, or the library's calls where `own`
    work(case)          bytes and operations one pass cannot do without
    exact(case, seed)   the same results in 64 bits

The cache: pages of `page` tokens; page p and KV head h hold E4M3 codes k, v [page, d] and one E8M0
exponent each (value = code 2^(e - 127)). A sequence's position x lies in page table[x // page], slot
x % page; an entry of -1 is no page. The operators ("op" of a case):
    attend   softmax(q k^T / sqrt(d)) v of the new tokens' query heads: a row at position p sees
             positions x <= p of its sequence with p - x < window or x < sinks
    select   beam search's step: of `b` prompts' `w` beams with logits [b w, v] the w best continuations,
             by the sum of log-probabilities
    reorder  the beams' page tables and lengths follow their parents in every layer's pool; a page that
             is being written has one owner, so its tokens are copied for a parent's further children
    copy     pages copied within every layer's pool
"""
from __future__ import annotations

import random

import torch

own = False


# ---------------------------------------------------------------- cases

QWEN = {"h": 14, "kv": 2, "d": 64}   # the 0.5B decoder
WIDE = {"h": 32, "kv": 8, "d": 128}  # a 7B-sized decoder with grouped queries


def listed() -> list[dict]:
    return [
        # one layer of a long chat's next token
        {"name": "step-1", "op": "attend", "b": 1, "past": 5000, "new": 1, "idle": 0, "pad": 0, "page": 16,
         "window": 1024, "sinks": 4, **QWEN},
        # 64 long conversations decoded together, some of the batch's places empty
        {"name": "step-64", "op": "attend", "b": 64, "past": 30000, "new": 1, "idle": 3, "pad": 3, "page": 32,
         "window": 4096, "sinks": 4, **WIDE},
        # a long prompt
        {"name": "prompt-2048", "op": "attend", "b": 1, "past": 0, "new": 2048, "idle": 0, "pad": 0, "page": 64,
         "window": 512, "sinks": 4, **WIDE},
        # a chunk of a document behind what is cached, a system prompt that stays visible, 16 heads on one
        {"name": "chunk-300", "op": "attend", "b": 1, "past": 9000, "new": 300, "idle": 0, "pad": 5, "page": 128,
         "window": 2000, "sinks": 130, "h": 16, "kv": 1, "d": 128},
        # prompts and steps in one call, a plain window
        {"name": "mixed-24", "op": "attend", "b": 24, "past": 1500, "new": 300, "idle": 1, "pad": 5, "page": 16,
         "window": 256, "sinks": 0, **QWEN},
        # a single prompt's beams
        {"name": "select-1x4", "op": "select", "b": 1, "w": 4, "v": 151936, "slack": 0, "done": 0, "masked": 0.0},
        # many prompts' beams, some of them finished
        {"name": "select-16x8", "op": "select", "b": 16, "w": 8, "v": 151936, "slack": 0, "done": 9, "masked": 0.0},
        # a vocabulary of an odd size, of which a grammar lets few tokens through
        {"name": "select-5x3", "op": "select", "b": 5, "w": 3, "v": 32003, "slack": 2, "done": 1, "masked": 0.9},
        # the state of a single prompt's beams in 24 layers
        {"name": "reorder-1x4", "op": "reorder", "b": 1, "w": 4, "past": 300, "layers": 24, "page": 32, "done": 0,
         **QWEN},
        # of several prompts' in 32 layers
        {"name": "reorder-8x5", "op": "reorder", "b": 8, "w": 5, "past": 1900, "layers": 32, "page": 64, "done": 3,
         **WIDE},
        # the pages that a forked conversation is about to write
        {"name": "copy-3", "op": "copy", "n": 3, "pages": 64, "layers": 24, "page": 16, **QWEN},
        # a pool compacted
        {"name": "copy-250", "op": "copy", "n": 250, "pages": 520, "layers": 16, "page": 32, **WIDE},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng) -> dict:
    op = rng.choice(["attend", "attend", "attend", "select", "select", "reorder", "copy"])
    if op == "select":
        b, w, v = _spread(rng, 1, 16), rng.choice([1, 2, 3, 4, 5, 8, 8, 13, 16, 32]), _spread(rng, 97, 200000)
        while b > 1 and b * w * v > 1.9e7:
            b = (b + 1) // 2
        while w > 1 and b * w * v > 1.9e7:
            w //= 2
        return {"op": op, "b": b, "w": w, "v": v, "slack": rng.choice([0, 0, 1, 6]),
                "done": rng.randrange(0, 1 + b * w // 4), "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}
    kv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "kv": kv, "h": kv * rng.choice([1, 2, 4, 7, 8, 16] if kv < 4 else [1, 2, 4, 7]),
            "d": rng.choice([32, 64, 64, 128, 128]), "page": rng.choice([16, 32, 64, 128])}
    if op == "copy":
        layers, n = _spread(rng, 1, 32), _spread(rng, 1, 250)
        while layers * n * kv * case["page"] * case["d"] > 1.3e8:
            n, layers = (n + 1) // 2, (layers + 1) // 2
        return {**case, "n": n, "pages": 2 * n + rng.randrange(0, 40), "layers": layers}
    if op == "reorder":
        b, w, layers = _spread(rng, 1, 12), rng.choice([1, 2, 3, 4, 5, 8, 11, 16, 32]), _spread(rng, 1, 32)
        while layers > 1 and b * w * layers * kv * case["page"] * case["d"] > 8e7:
            b, layers = (b + 1) // 2, (layers + 1) // 2
        return {**case, "b": b, "w": w, "past": _spread(rng, 1, 3000), "layers": layers,
                "done": rng.randrange(0, 1 + b * w // 4)}
    case["window"], case["sinks"] = _spread(rng, 1, 6000), rng.choice([0, 0, 1, 4, 4, 64, 200])
    if rng.random() < 0.5:  # steps
        b, past, new = _spread(rng, 1, 64), _spread(rng, 1, 40000), 1
    elif rng.random() < 0.4:  # a prompt or a chunk of one
        b, past, new = 1, rng.choice([0, 0, _spread(rng, 1, 12000)]), _spread(rng, 2, 2048)
    else:  # several prompts, or prompts and steps
        b, past, new = _spread(rng, 2, 24), _spread(rng, 1, 3000), _spread(rng, 2, 700)
    seen = lambda: case["sinks"] + min(past + new, case["window"])  # noqa: E731
    while b > 1 and (b * case["h"] * new * seen() > 3e7 or b * (seen() + new) * kv * case["d"] > 2.6e8):
        b = (b + 1) // 2
    while case["h"] * new * seen() > 3e7:
        new = new // 2
    return {**case, "b": b, "past": past, "new": new, "idle": rng.randrange(0, 1 + b // 8), "pad": rng.choice([0, 0, 7])}


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Cached and new tokens of each sequence: the first has `past` and `new`, the others fewer, the last
    `idle` of them no new token."""
    b, past, new = case["b"], case["past"], case["new"]
    rng = random.Random(b * 8191 + past + 31 * new)
    pasts = [past] + [int(past * rng.uniform(0.02, 1.0)) for _ in range(b - 1)]
    news = [new] + [1 if rng.random() < 0.5 else rng.randint(1, new) for _ in range(b - 1)]
    return pasts, [0 if i >= b - case["idle"] else n for i, n in enumerate(news)]


def _family(case: dict) -> tuple[list[int], list[int], list[int]]:
    """Of a reorder's places: tokens held before the last pass, parent (a place of the same prompt) and
    whether the beam is done. Good beams have several children and others none."""
    b, w, past = case["b"], case["w"], case["past"]
    rng = random.Random(b * 8191 + w * 127 + past)
    pasts, parent = [], []
    for g in range(b):
        pasts += [past if g == 0 else int(past * rng.uniform(0.3, 1.0))] * w
        parent += [g * w + min(rng.randrange(w), rng.randrange(w)) for _ in range(w)]
    done = set(rng.sample(range(b * w), case["done"]))
    return pasts, parent, [int(i in done) for i in range(b * w)]


def _live(case: dict) -> int:
    """Rows of logits that a selection reads."""
    return case["b"] * case["w"] - case["done"]


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
    """(E4M3 codes uint8, E8M0 exponents uint8) of x [.., page, d]."""
    e = _e8m0(x.abs().amax((-2, -1)))
    codes = (x * _pow2(254 - e.int())[..., None, None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), e


def _pool(case: dict, pages: int, rnd, gain=1.0) -> dict:
    """The pools of every layer: codes [layers, pages, kv, page, d], exponents [layers, pages, kv]."""
    kv, d, page, layers = case["kv"], case["d"], case["page"], case.get("layers", 1)
    blocks = [(_blocks(rnd(pages, kv, page, d) * gain),
               _blocks(rnd(pages, kv, page, d) * torch.exp2(2 * rnd(pages, 1, page, 1)))) for _ in range(layers)]
    return {n: torch.stack([x[i][j] for x in blocks]) for n, i, j in (("k", 0, 0), ("ke", 0, 1), ("v", 1, 0),
                                                                     ("ve", 1, 1))}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    order = lambda n: torch.randperm(n, generator=g, device="cuda").to(torch.int32)  # noqa: E731
    return {"case": case, **{"attend": _attend_inputs, "select": _select_inputs, "reorder": _reorder_inputs,
                             "copy": _copy_inputs}[case["op"]](case, rnd, order)}


def _attend_inputs(case: dict, rnd, order) -> dict:
    h, kv, d, page, b = case["h"], case["kv"], case["d"], case["page"], case["b"]
    pasts, news = _lengths(case)
    n, wide = sum(news), max(-(-(p + m) // page) for p, m in zip(pasts, news)) + 1
    table = torch.full((b, wide), -1, dtype=torch.int32)
    # pages wholly behind the window have been given back
    held = [[j for j in range(-(-(p + m) // page))
             if j * page < case["sinks"] or (j + 1) * page > p - case["window"] + 1] for p, m in zip(pasts, news)]
    pages = sum(map(len, held)) + 3
    ids, at = order(pages).cpu(), 0  # handed out in no order
    for i, js in enumerate(held):
        table[i, js] = ids[at:at + len(js)]
        at += len(js)
    gain = torch.where(rnd(kv, 1, d) > 1.5, 6.0, 1.0)  # keys' large channels
    starts = torch.tensor([sum(news[:i]) for i in range(b + 1)], dtype=torch.int32)
    t = n + case["pad"]
    return {"n": n, "t": t, "max_new": max(news), "table": table.cuda(), "q_start": starts.cuda(),
            "past": torch.tensor(pasts, dtype=torch.int32).cuda(), "pool": _pool(case, pages, rnd, gain),
            "q": rnd(t, h * d) * 1.5, "out": rnd(t, h * d)}


def _select_inputs(case: dict, rnd, order) -> dict:
    b, w, v = case["b"], case["w"], case["v"]
    # a few tokens far above the rest, as a trained model's logits; beams differ in how sure they are
    x = rnd(b * w, v + case["slack"]) * (1.5 + 0.5 * rnd(b * w, 1).abs())
    x += 9.0 * (rnd(b * w, v + case["slack"]) > 3.6) * rnd(b * w, 1).abs()
    if case["masked"]:
        x[rnd(b * w, v + case["slack"]).abs() > _quantile(1 - case["masked"])] = float("-inf")
    score = -30.0 + 6.0 * rnd(b * w)
    done = torch.zeros(b * w, dtype=torch.int32, device="cuda")
    done[order(b * w)[:case["done"]].long()] = 1
    new = lambda dt: torch.zeros(b * w, dtype=dt, device="cuda")  # noqa: E731
    return {"logits": x, "score": score, "done": done, "eos": int(order(v)[0]), "tok": new(torch.int32),
            "parent": new(torch.int32), "new_score": new(torch.float32), "new_done": new(torch.int32)}


def _quantile(p: float) -> float:
    """|x| of a standard normal that a share p lies below."""
    return 2 ** 0.5 * float(torch.erfinv(torch.tensor(p, dtype=torch.float64)))


def _reorder_inputs(case: dict, rnd, order) -> dict:
    b, w, page = case["b"], case["w"], case["page"]
    pasts, parent, done = _family(case)
    rows, wide = b * w, max(pasts) // page + 2
    pages = 2 * rows + 5  # of the pages being written and the next; earlier ones are only named
    ids = order(pages).cpu()
    table = torch.full((rows, wide), -1, dtype=torch.int32)
    mine = torch.full((rows, wide), -1, dtype=torch.int32)
    shuffled = torch.argsort(rnd(b, w), 1).cpu()
    for i in range(rows):
        at, g = pasts[i] // page, i // w
        table[i, :at] = torch.arange(at, dtype=torch.int32) % pages
        mine[i, at:at + 2] = ids[2 * i:2 * i + 2][:wide - at]
        table[i, at] = ids[2 * (g * w + int(shuffled[g, i % w]))]  # an earlier order's
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    return {"past": i32(pasts), "parent": i32(parent), "done": i32(done), "table": table.cuda(), "own": mine.cuda(),
            "new_table": torch.zeros_like(table).cuda(), "new_past": i32([0] * rows),
            "pool": _pool(case, pages, rnd)}


def _copy_inputs(case: dict, rnd, order) -> dict:
    ids = order(case["pages"])
    return {"src": ids[:case["n"]].contiguous(), "dst": ids[case["n"]:2 * case["n"]].contiguous(),
            "pool": _pool(case, case["pages"], rnd)}


# ---------------------------------------------------------------- the plain forms

def _rows(s: dict):
    """Sequence and place in it of each new token."""
    rows = torch.arange(s["n"], device="cuda", dtype=torch.int32)
    seq = torch.bucketize(rows, s["q_start"][1:], right=True)
    return seq, rows - s["q_start"][seq]


def _plain_attend(s: dict):
    c, pool = s["case"], {n: x[0] for n, x in s["pool"].items()}
    h, kv, d, new, b, page = c["h"], c["kv"], c["d"], s["max_new"], c["b"], c["page"]
    # positions that some row of a sequence may see: the sinks, then from the first row's window on
    past, wide = s["past"].long(), s["table"].shape[1] * page
    sinks = min(c["sinks"], wide)
    span = min(wide, c["window"] + new)
    first = (past - c["window"] + 1).clamp(min=sinks)
    pos = torch.cat([torch.arange(sinks, device="cuda").expand(b, -1),
                     first[:, None] + torch.arange(span, device="cuda")], 1)
    at = pos.clamp(max=wide - 1)
    pg = s["table"].gather(1, at // page)
    row = (pg.clamp(min=0).long(), slice(None), at % page)

    def held(codes, e):
        x = codes[row].view(torch.float8_e4m3fn).float() * _pow2(e[pg.clamp(min=0).long()])[..., None]
        return x.transpose(1, 2)  # [b, kv, keys, d]

    k, v = held(pool["k"], pool["ke"]), held(pool["v"], pool["ve"])
    q = s["q"][(s["q_start"][:-1, None] + torch.arange(new, device="cuda")).clamp(max=s["t"] - 1)]
    q = q.reshape(b, new, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)
    sc = (q @ k.transpose(2, 3).contiguous() / d ** 0.5).reshape(b, kv, new, -1, pos.shape[1])
    p = (past[:, None] + torch.arange(new, device="cuda"))[:, :, None]
    x = pos[:, None]
    seen = (x <= p) & ((p - x < c["window"]) | (x < sinks)) & (pg >= 0)[:, None]
    sc = sc.masked_fill(~seen[:, None, :, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    w = torch.exp(sc - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    l = w.sum(-1, keepdim=True)
    o = (w.reshape(b, kv, -1, pos.shape[1]) @ v.contiguous()).reshape(w.shape[:-1] + (d,))
    o = o / torch.where(l > 0, l, torch.ones_like(l))
    seq, i = _rows(s)
    s["out"][:s["n"]] = o.permute(0, 2, 1, 3, 4).reshape(b, new, h * d)[seq, i]


def _plain_select(s: dict):
    c = s["case"]
    b, w, v = c["b"], c["w"], c["v"]
    x = s["logits"][:, :v]
    m = x.amax(1, keepdim=True)
    lse = m[:, 0].double() + torch.exp(x - m).sum(1).double().log()
    # one column more: a done beam as it is
    none = torch.full((b * w, 1), float("-inf"), dtype=torch.float64, device="cuda")
    done = (s["done"] != 0)[:, None]
    cand = torch.cat([torch.where(done, none, s["score"].double()[:, None] + (x.double() - lse[:, None])),
                      torch.where(done, s["score"].double()[:, None], none)], 1)
    cand = torch.where(cand.isnan(), none, cand).reshape(b, w * (v + 1))
    at = torch.arange(cand.shape[1], device="cuda")
    group = torch.arange(b, device="cuda")
    for i in range(w):
        best = cand.amax(1)
        flat = torch.where(cand == best[:, None], at, cand.shape[1]).amin(1)  # the first of equals
        some = best > float("-inf")
        beam, tok = flat // (v + 1), flat % (v + 1)
        place = group * w + i
        s["parent"][place] = torch.where(some, group * w + beam, -1).int()
        s["tok"][place] = torch.where(some & (tok < v), tok, s["eos"]).int()
        s["new_score"][place] = best.float()
        s["new_done"][place] = (some & ((tok == v) | (tok == s["eos"]))).int()
        cand[group, flat] = float("-inf")


def _plain_reorder(s: dict):
    c = s["case"]
    b, w, page = c["b"], c["w"], c["page"]
    rows = b * w
    at = torch.arange(rows, device="cuda")
    parent = s["parent"].long()
    goes_on = (parent >= 0) & (s["done"] == 0)
    p = parent.clamp(min=0)
    length = torch.where(goes_on, s["past"][p] + 1, -1)
    tail, used = (length.clamp(min=0) // page).long(), length.clamp(min=0) % page
    column = torch.arange(s["table"].shape[1], device="cuda")
    table = torch.where(column < tail[:, None], s["table"][p], s["own"])
    copied = goes_on & (used > 0)
    was = s["table"][p, tail]  # the parent's page that is being written
    same = (p[:, None] == p) & copied[:, None] & copied
    first = copied & ~(same & (at < at[:, None])).any(1)
    # the others of a group take its pages that no first child keeps, in their order
    group = at // w
    together = (group[:, None] == group) & (tail[:, None] == tail)
    more = copied & ~first
    rank = (more[None] & more[:, None] & together & (at < at[:, None])).sum(1)
    spare = s["own"][:, tail].t().reshape(rows, b, w)[at, group]  # [row, places of its group]: pages at its tail
    kept = torch.where(first, was, -2).reshape(b, w)[group]
    free = (spare >= 0) & ~(spare[:, :, None] == kept[:, None]).any(2)
    nth = free.long().cumsum(1) - 1
    pick = (free & (nth == rank[:, None])).long()
    mine = torch.where(first, was, (spare * pick).sum(1).int())
    s["new_table"].copy_(torch.where(goes_on[:, None], torch.where(
        copied[:, None] & (column == tail[:, None]), mine[:, None], table), -1))
    s["new_past"].copy_(length)
    # places without a copy write a page that none of the others takes, as it is
    pages = s["pool"]["k"].shape[1]
    taken = torch.zeros(pages + 1, device="cuda").index_fill_(0, torch.where(more, mine.long(), pages), 1.0)
    idle = taken[:pages].argmin()
    src, dst = torch.where(more, was.long(), idle), torch.where(more, mine.long(), idle)
    slot = ((torch.arange(page, device="cuda") < used[:, None]) & more[:, None])[:, None, :, None]
    for n in ("k", "v"):
        x, e = s["pool"][n], s["pool"][n + "e"]
        x[:, dst] = torch.where(slot, x[:, src], x[:, dst])
        e[:, dst] = torch.where(more[:, None], e[:, src], e[:, dst])


def _plain_copy(s: dict):
    src, dst = s["src"].long(), s["dst"].long()
    for x in s["pool"].values():
        x[:, dst] = x[:, src]


PLAIN = {"attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder, "copy": _plain_copy}


# ---------------------------------------------------------------- the library's calls

def _handle(s: dict):
    """The argument structures and the workspace that a program keeps between calls."""
    import ctypes as C

    from lowbit_amd import kernels as K
    c, L, ptr = s["case"], K.lib(), lambda t: t.data_ptr()  # noqa: E731
    stream, space = torch.cuda.current_stream().cuda_stream, lambda n: torch.empty(  # noqa: E731
        max(256, n), dtype=torch.uint8, device="cuda")
    if c["op"] == "select":
        beams = K.LbdBeams(ptr(s["score"]), ptr(s["done"]), ptr(s["new_score"]), ptr(s["new_done"]), ptr(s["tok"]),
                           ptr(s["parent"]), None, None, None, 0, c["b"], c["w"], c["v"], s["eos"])
        need = L.lbd_beam_select_work_bytes(C.byref(beams))
        ws = space(need)
        args = ptr(s["logits"]), s["logits"].shape[1], C.byref(beams), ptr(ws), need, stream
        return L.lbd_beam_select, args, K._check, (beams, ws)
    layers, pages = s["pool"]["k"].shape[:2]
    pools = (K.LbdKv8Pool * layers)(*(
        K.LbdKv8Pool(*(ptr(s["pool"][n][i]) for n in ("k", "v", "ke", "ve")), pages, c["page"], c["kv"], c["d"])
        for i in range(layers)))
    if c["op"] == "copy":
        return L.lbd_kv8_copy_pages, (pools, layers, ptr(s["src"]), ptr(s["dst"]), c["n"], stream), K._check, pools
    if c["op"] == "reorder":
        order = K.LbdKv8Order(ptr(s["parent"]), ptr(s["done"]), ptr(s["past"]), ptr(s["table"]), ptr(s["own"]),
                              ptr(s["new_past"]), ptr(s["new_table"]), c["b"], c["w"], s["table"].shape[1], 1)
        return L.lbd_kv8_reorder, (pools, layers, C.byref(order), stream), K._check, (pools, order)
    batch = K.LbdKv8Batch(ptr(s["q_start"]), ptr(s["past"]), ptr(s["table"]), c["b"], s["table"].shape[1], s["max_new"],
                          s["t"])
    need = L.lbd_kv8_attention_window_work_bytes(C.byref(pools[0]), C.byref(batch), c["h"], c["window"], c["sinks"])
    ws = space(need)
    args = (C.byref(pools[0]), C.byref(batch), ptr(s["q"]), c["h"] * c["d"], c["h"], c["window"], c["sinks"],
            ptr(s["out"]), c["h"] * c["d"], ptr(ws), need, stream)
    return L.lbd_kv8_attention_window, args, K._check, (pools, batch, ws)


def run(s: dict):
    if own:
        if "handle" not in s:
            s["handle"] = _handle(s)
        fn, args, check, _ = s["handle"]
        check(fn(*args), s["case"]["op"], False)
    else:
        PLAIN[s["case"]["op"]](s)
    if s["case"]["op"] == "attend":
        return s["out"]
    if s["case"]["op"] == "select":
        return {n: s[n] for n in ("tok", "parent", "new_score", "new_done")}
    held = {n: x.view(torch.float8_e4m3fn if len(n) == 1 else torch.float8_e8m0fnu) for n, x in s["pool"].items()}
    return held if s["case"]["op"] == "copy" else {"table": s["new_table"], "past": s["new_past"], **held}


# ---------------------------------------------------------------- work

def _copies(case: dict) -> list[int]:
    """Tokens of each page that a reorder copies."""
    pasts, parent, done = _family(case)
    kept, out = set(), []
    for p, d in zip(parent, done):
        used = (pasts[p] + 1) % case["page"]
        if d or not used:
            continue
        if p in kept:
            out.append(used)
        kept.add(p)
    return out


def work(case: dict) -> dict:
    if case["op"] == "select":
        n = _live(case) * case["v"]
        return {"bytes": 4 * n + 24 * case["b"] * case["w"], "flops": 4 * n}
    h, kv, d, page = case["h"], case["kv"], case["d"], case["page"]
    if case["op"] == "copy":
        return {"bytes": case["layers"] * case["n"] * 2 * kv * (2 * page * d + 2) + 8 * case["n"], "flops": 0}
    if case["op"] == "reorder":
        pasts, parent, done = _family(case)
        columns = sum(pasts[p] // page + 1 for p, d_ in zip(parent, done) if not d_)
        return {"bytes": case["layers"] * 2 * kv * sum(2 * u * d + 2 for u in _copies(case)) + 8 * columns
                + 20 * case["b"] * case["w"], "flops": 0}
    pasts, news = _lengths(case)
    win, sinks, n = case["window"], case["sinks"], sum(news)
    keys = pairs = 0
    for p, m in zip(pasts, news):
        if not m:
            continue
        first = max(0, p - win + 1)
        keys += p + m - first + min(sinks, first)
        pairs += sum(min(x + 1, win) + min(sinks, max(0, x + 1 - win)) for x in range(p, p + m))
    return {"bytes": 8 * n * h * d + 2 * kv * keys * (d + 1 / page), "flops": 4 * pairs * h * d}


# ---------------------------------------------------------------- the results in 64 bits

def _values(codes: torch.Tensor) -> torch.Tensor:
    """float64 that E4M3 bytes stand for."""
    man, ex = [c & 7 for c in range(256)], [(c >> 3) & 15 for c in range(256)]
    x = [(8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9 for m, e in zip(man, ex)]
    x = [-y if c > 127 else y for c, y in enumerate(x)]
    return torch.tensor(x, dtype=torch.float64, device="cuda")[codes.long()]


def _scales(e: torch.Tensor) -> torch.Tensor:
    """float64 2^(e - 127) of E8M0 bytes."""
    return torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=torch.float64, device="cuda")[e.long()]


def _exact_attend(s: dict):
    c, pool = s["case"], {n: x[0] for n, x in s["pool"].items()}
    h, kv, d, page = c["h"], c["kv"], c["d"], c["page"]
    out, row, (pasts, news) = s["out"].double(), 0, _lengths(c)
    table = s["table"].cpu().tolist()
    for b, (past, new) in enumerate(zip(pasts, news)):
        if not new:
            continue
        # the held pages, the positions that they hold and, row by row, which of them are seen
        js = [j for j in range(-(-(past + new) // page)) if table[b][j] >= 0]
        pages = torch.tensor([table[b][j] for j in js], device="cuda")
        pos = (torch.tensor(js, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
        k, v = ((_values(pool[n][pages]) * _scales(pool[n + "e"][pages])[:, :, None, None]).transpose(0, 1).reshape(
            kv, -1, d) for n in "kv")
        mine = past + torch.arange(new, device="cuda")[:, None]
        hidden = (pos > mine) | ((pos <= mine - c["window"]) & (pos >= c["sinks"]))
        for j in range(h):
            q = s["q"][row:row + new, j * d:(j + 1) * d].double()
            sc = (q @ k[j // (h // kv)].t() / d ** 0.5).masked_fill(hidden, float("-inf"))
            out[row:row + new, j * d:(j + 1) * d] = torch.softmax(sc, 1) @ v[j // (h // kv)]
        row += new
    return out


def _exact_select(s: dict):
    c = s["case"]
    b, w, v = c["b"], c["w"], c["v"]
    out = {"tok": [], "parent": [], "new_score": [], "new_done": []}
    done, score = s["done"].cpu().tolist(), s["score"].double().cpu().tolist()
    for g in range(b):
        cand = []  # (sum, beam, place among the beam's, token, done)
        for i in range(g * w, g * w + w):
            if done[i]:
                cand.append((score[i], i, 0, s["eos"], 1))
                continue
            logp = torch.log_softmax(s["logits"][i, :v].double(), 0)
            val, tok = torch.sort(logp, descending=True, stable=True)
            cand += [(score[i] + x, i, n, t, int(t == s["eos"]))
                     for n, (x, t) in enumerate(zip(val[:w].tolist(), tok[:w].tolist())) if x > float("-inf")]
        cand.sort(key=lambda x: (-x[0], x[1], x[2]))
        cand = cand[:w] + [(float("-inf"), -1, 0, s["eos"], 0)] * (w - len(cand))
        for n, j in (("new_score", 0), ("parent", 1), ("tok", 3), ("new_done", 4)):
            out[n] += [x[j] for x in cand]
    return {n: torch.tensor(x, dtype=torch.float64 if n == "new_score" else torch.int32, device="cuda")
            for n, x in out.items()}


def _moved(s: dict, moves) -> dict:
    """The pools' values after (source, destination, tokens) of `moves`, in 64 bits."""
    out = {n: _values(x) if len(n) == 1 else _scales(x) for n, x in s["pool"].items()}
    for a, b, n in moves:
        for x in (out["k"], out["v"]):
            x[:, b, :, :n] = x[:, a, :, :n]
        for x in (out["ke"], out["ve"]):
            x[:, b] = x[:, a]
    return out


def _exact_reorder(s: dict):
    c = s["case"]
    b, w, page = c["b"], c["w"], c["page"]
    pasts, parent, done = _family(c)
    table, mine = s["table"].cpu().tolist(), s["own"].cpu().tolist()
    new_table, new_past, moves = [[-1] * len(table[0]) for _ in table], [-1] * len(table), []
    for g in range(b):
        places = range(g * w, g * w + w)
        heir = {}
        for i in places:
            if not done[i]:
                heir.setdefault(parent[i], i)
        taken = {table[p][(pasts[p] + 1) // page] for p in heir if (pasts[p] + 1) % page}
        spare = {}
        for i in places:
            if done[i]:
                continue
            p = parent[i]
            at, used = divmod(pasts[p] + 1, page)
            new_past[i] = pasts[p] + 1
            new_table[i] = table[p][:at] + mine[i][at:]
            if used and heir[p] == i:
                new_table[i][at] = table[p][at]
            elif used:
                left = spare.setdefault(at, [mine[j][at] for j in places if mine[j][at] not in taken])
                new_table[i][at] = left.pop(0)
                moves.append((table[p][at], new_table[i][at], used))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"table": i32(new_table), "past": i32(new_past), **_moved(s, moves)}


def _exact_copy(s: dict):
    return _moved(s, [(a, b, s["case"]["page"]) for a, b in zip(s["src"].tolist(), s["dst"].tolist())])


def exact(case: dict, seed: int):
    return {"attend": _exact_attend, "select": _exact_select, "reorder": _exact_reorder, "copy": _exact_copy}[case["op"]](
        prepare(case, seed))
