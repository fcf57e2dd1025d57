"""The operators of the token stage on an 8-bit paged cache, with their plain forms and the cases they are timed at.

The pixel decoder's input is a sequence of visual tokens that a language model draws one at a time.  Four operators
serve that loop: `page_advance` keeps the block tables, `cache_write` stores keys and values in 8 bits,
`cached_attention` reads them, `sample_tokens` draws the next ids.  With `own = False`, `run` computes them in
elementary torch operations; with `own = True` it calls `pigeon_amd.ops`.

Cache layout (P tokens to a page, one power-of-two scale per page and head):
  k_pages e4m3 [pages, kv_heads, P, D]     v_pages e4m3 [pages, kv_heads, D, P]     scales fp32 [pages, kv_heads]
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCAB = 32002 + 16384          # text ids and specials, then the codebook's ids
SCALE_FLOOR = -100             # smallest scale of a page: 2^-100


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a full batch: every request gets one token, a page once in a while
        {"name": "pages_decode_b64", "op": "pages", "R": 64, "P": 16, "held": 2048, "add": 1, "T": 64, "shape": 1},
        # a step that finishes requests, rolls some back and admits long prompts
        {"name": "pages_prompts_b512", "op": "pages", "R": 512, "P": 64, "held": 4096, "add": 1000, "T": 524288, "shape": 2},
        # the decoding step's own keys and values: one token a request
        {"name": "write_decode_b64", "op": "write", "T": 64, "R": 64, "H": 32, "D": 128, "P": 16, "dtype": "bf16", "shape": 3},
        # ragged prompts, grouped heads
        {"name": "write_prompts_16k", "op": "write", "T": 16384, "R": 13, "H": 8, "D": 128, "P": 64, "dtype": "fp16", "shape": 4},
        # one request, short cache: latency
        {"name": "decode_b1_l257", "op": "attend", "R": 1, "Hq": 32, "Hkv": 32, "D": 128, "P": 16, "len_lo": 257, "len_hi": 257,
         "q_lo": 1, "q_hi": 1, "window": 0, "dtype": "bf16", "shape": 5},
        # a batch in mid-conversation, one head per query head, ragged lengths
        {"name": "decode_b16_l4k", "op": "attend", "R": 16, "Hq": 32, "Hkv": 32, "D": 128, "P": 16, "len_lo": 900, "len_hi": 4096,
         "q_lo": 1, "q_hi": 1, "window": 0, "dtype": "bf16", "shape": 6},
        # few long requests, grouped heads: the long axis has to be split
        {"name": "decode_b4_l128k_gqa", "op": "attend", "R": 4, "Hq": 32, "Hkv": 8, "D": 128, "P": 64, "len_lo": 60000, "len_hi": 131072,
         "q_lo": 1, "q_hi": 1, "window": 0, "dtype": "fp16", "shape": 7},
        # chunks of prompts against what is cached: a large matrix product
        {"name": "prompt_b4_n2k", "op": "attend", "R": 4, "Hq": 32, "Hkv": 32, "D": 128, "P": 16, "len_lo": 2048, "len_hi": 8192,
         "q_lo": 2048, "q_hi": 2048, "window": 0, "dtype": "bf16", "shape": 8},
        # ragged chunks and single tokens in one call, narrow heads, a sliding window
        {"name": "mixed_b24_window", "op": "attend", "R": 24, "Hq": 16, "Hkv": 4, "D": 64, "P": 32, "len_lo": 40, "len_hi": 6000,
         "q_lo": 1, "q_hi": 700, "window": 1024, "dtype": "fp16", "shape": 9},
        # one request's next token
        {"name": "sample_b1", "op": "sample", "B": 1, "V": VOCAB, "dtype": "fp32", "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # a batch, with every filter
        {"name": "sample_b64_k50", "op": "sample", "B": 64, "V": VOCAB, "dtype": "bf16", "top_k": 50, "top_p": 0.95, "min_p": 0.01},
        # a large batch over a large vocabulary, nucleus only
        {"name": "sample_b256_v128k", "op": "sample", "B": 256, "V": 131072, "dtype": "bf16", "top_k": 0, "top_p": 0.92, "min_p": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "write", "attend", "attend", "sample"])
    shape = rng.randrange(1 << 30)
    if op == "pages":
        R, add = _log_int(rng, 1, 700), rng.choice([1, 1, _log_int(rng, 2, 700)])
        return {"op": op, "R": R, "P": rng.choice([16, 32, 64, 128]), "held": _log_int(rng, 1, 4096), "add": add, "T": R * add, "shape": shape}
    if op == "write":
        R = _log_int(rng, 1, 100)
        return {"op": op, "T": R * rng.choice([1, _log_int(rng, 1, 80)]), "R": R, "H": rng.choice([1, 2, 4, 5, 8]), "D": rng.choice([64, 128, 256]),
                "P": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"]), "shape": shape}
    if op == "sample":
        return {"op": op, "B": _log_int(rng, 1, 250), "V": _log_int(rng, 1000, 130000), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "top_k": rng.choice([0, 0, 1, _log_int(rng, 2, 900)]), "top_p": rng.choice([1.0, 0.5, 0.9, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.02])}
    G, Hkv = rng.choice([(1, 8), (1, 16), (1, 32), (2, 8), (4, 4), (4, 8), (5, 2), (7, 4), (8, 2), (8, 8), (16, 1)])
    case = {"op": op, "Hq": G * Hkv, "Hkv": Hkv, "D": rng.choice([64, 128, 128, 256]), "P": rng.choice([16, 32, 64, 128]),
            "window": rng.choice([0, 0, 0, _log_int(rng, 16, 2000)]), "dtype": rng.choice(["bf16", "fp16"]), "shape": shape}
    if rng.random() < 0.6:                                      # single tokens
        R = _log_int(rng, 1, 64)
        hi = _log_int(rng, 16, 100000 // R + 2000)
        return {**case, "R": R, "len_lo": max(1, hi // rng.choice([1, 3, 20])), "len_hi": hi, "q_lo": 1, "q_hi": 1}
    R = _log_int(rng, 1, 12)                                    # prompts, whole or in chunks
    hi = _log_int(rng, 2, 6000 // R + 200)
    q = max(1, hi // rng.choice([1, 1, 2, 8]))
    return {**case, "R": R, "len_lo": max(1, hi // 4), "len_hi": hi, "q_lo": max(1, q // 8), "q_hi": q}


# ---------------------------------------------------------------------------------------------------- sizes of a case
def _lengths(case):
    """Held lengths and queries of each request of an attention case (sizes depend on the case alone, values on the seed)."""
    r = random.Random(case["shape"])
    lens = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["R"])]
    return lens, [min(n, r.randint(case["q_lo"], case["q_hi"])) for n in lens]


def _page_lengths(case):
    r = random.Random(case["shape"])
    R, held = case["R"], [r.randint(0, case["held"]) for _ in range(case["R"])]
    if case["add"] == 1:                                        # decoding: all held tokens stay, one is added
        return held, list(held), [1] * R
    keep = [r.choice([0, h, h, max(0, h - 3)]) for h in held]   # finished, going on, rolled back
    return held, keep, [r.randint(0, case["add"]) for _ in range(R)]


def _write_lengths(case):
    """Tokens that each request held before the call, and how many it writes (they sum to T)."""
    r = random.Random(case["shape"])
    R, T = case["R"], case["T"]
    cuts = sorted(r.randint(0, T - R) for _ in range(R - 1))
    new = [b - a + 1 for a, b in zip([0] + cuts, cuts + [T - R])]
    return [r.randint(0, 4 * case["P"]) for _ in range(R)], new


def _pairs(case):
    """Query-key pairs that the masks leave, per head, and the keys that any query of a request sees."""
    pairs = keys = 0
    for L, n in zip(*_lengths(case)):
        w = case["window"] or L
        pairs += sum(min(p + 1, w) for p in range(L - n, L))
        keys += min(L, n + w - 1)
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "pages":
        held, keep, add = _page_lengths(case)
        P = case["P"]
        moved = sum(-(-h // P) + -(-(k + a) // P) - 2 * -(-k // P) for h, k, a in zip(held, keep, add))
        return {"bytes": 8 * case["T"] + 8 * moved + 24 * case["R"], "flops": 0}
    if op == "write":
        return {"bytes": case["T"] * (2 * case["H"] * case["D"] * 3 + 8), "flops": 4 * case["T"] * case["H"] * case["D"]}
    if op == "sample":
        return {"bytes": case["B"] * (case["V"] * DTYPES[case["dtype"]].itemsize + 28), "flops": 4 * case["B"] * case["V"]}
    pairs, keys = _pairs(case)
    tokens = sum(_lengths(case)[1])
    return {"bytes": 2 * keys * case["Hkv"] * case["D"] + 4 * tokens * case["Hq"] * case["D"], "flops": 4 * pairs * case["Hq"] * case["D"]}


# ---------------------------------------------------------------------------------------------------- inputs
def _tables(lens, P, extra, g):
    """Disjoint pages for the given lengths out of a shuffled pool: (block table, pages left over in the order a stack gives them)."""
    need = [-(-n // P) for n in lens]
    W = max(1, max(need) + extra)
    pool = torch.randperm(sum(need) + extra * len(lens) // 4 + 3, generator=g, dtype=torch.int64).to(torch.int32)
    at = torch.tensor([0] + need).cumsum(0)
    col = torch.arange(W)
    idx = at[:-1, None] + col
    table = torch.where(col < torch.tensor(need)[:, None], pool[idx.clamp(max=len(pool) - 1)], -1).to(torch.int32)
    return table, pool[at[-1]:], len(pool)


def _pages(shape, g):
    """8-bit pages as a cache holds them: normal values of a size that differs by head, over their page's scale."""
    exp = torch.randint(-8, -4, shape[:2], generator=g, device=DEV)
    values = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(64).clamp_(-448, 448)
    return values.to(torch.float8_e4m3fn), torch.ldexp(torch.ones(shape[:2], device=DEV), exp)


def prepare(case, seed):
    op = case["op"]
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                                       # noqa: E731
    s = {"case": case}
    if op == "pages":
        held, keep, add = _page_lengths(case)
        P = case["P"]
        table, left, pages = _tables(held, P, -(-case["add"] // P) + 1, cpu)
        free = torch.zeros(pages, dtype=torch.int32)
        free[:len(left)] = left
        s |= {"lens": i32(held), "keep": i32(keep), "add": i32(add), "table": table.to(DEV), "free": free.to(DEV),
              "count": i32([len(left)]), "T": case["T"], "P": P}
    elif op == "write":
        held, new = _write_lengths(case)
        P, H, D = case["P"], case["H"], case["D"]
        table, _, pages = _tables([h + n for h, n in zip(held, new)], P, 0, cpu)
        rows = table.tolist()
        slots = [rows[r][p // P] * P + p % P for r in range(case["R"]) for p in range(held[r], held[r] + new[r])]
        s["k_pages"], s["k_scale"] = _pages((pages, H, P, D), g)
        s["v_pages"], s["v_scale"] = _pages((pages, H, D, P), g)
        size = torch.ldexp(torch.ones(H, 1, device=DEV), torch.arange(H, device=DEV)[:, None] % 4 - 1)
        # keys and values as a fused projection leaves them: [T, 2, H, D], so each has a stride of its own
        kv = (torch.randn(case["T"], 2, H, D, generator=g, device=DEV) * size).to(DTYPES[case["dtype"]])
        starts = torch.tensor([0] + new).cumsum(0)
        s |= {"k": kv[:, 0], "v": kv[:, 1], "slots": torch.tensor(slots, dtype=torch.int64, device=DEV), "starts": i32(starts.tolist())}
    elif op == "attend":
        lens, new = _lengths(case)
        P, D, dt = case["P"], case["D"], DTYPES[case["dtype"]]
        table, _, pages = _tables(lens, P, 0, cpu)
        s["k_pages"], s["k_scale"] = _pages((pages, case["Hkv"], P, D), g)
        s["v_pages"], s["v_scale"] = _pages((pages, case["Hkv"], D, P), g)
        starts = torch.tensor([0] + new).cumsum(0)
        s |= {"q": torch.randn(sum(new), case["Hq"], D, generator=g, device=DEV).to(dt), "table": table.to(DEV), "lens": i32(lens),
              "starts": None if case["q_hi"] == 1 else i32(starts.tolist()), "most": max(new)}
    else:
        B, V = case["B"], case["V"]
        # a few likely ids over a broad floor, as a trained model's logits are
        logits = torch.randn(B, V, generator=g, device=DEV) * 2
        logits += 9 * torch.rand(B, V, generator=g, device=DEV).pow_(40)
        logits[:, V // 3:V // 3 + V // 8] = -math.inf               # ids that may not be drawn here
        s |= {"logits": logits.to(DTYPES[case["dtype"]]), "u": torch.rand(B, generator=g, device=DEV),
              "temperature": torch.rand(B, generator=g, device=DEV) * 0.9 + 0.4,
              "top_k": torch.full((B,), case["top_k"], dtype=torch.int32, device=DEV),
              "top_p": torch.full((B,), case["top_p"], device=DEV), "min_p": torch.full((B,), case["min_p"], device=DEV)}
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_pages(s):
    P, T, table, free, count = s["P"], s["T"], s["table"], s["free"], s["count"]
    R, W = table.shape
    N = free.numel()
    held = s["lens"].long()
    keep = torch.minimum(s["keep"].long().clamp(min=0), held)
    n = s["add"].long().clamp(min=0)
    have, kept = (held + P - 1) // P, (keep + P - 1) // P
    col = torch.arange(W, device=DEV)
    dump = torch.full((), N, device=DEV)                               # where what has no place goes
    stack = torch.cat([free, free.new_zeros(1)])
    freed = have - kept
    back = freed.cumsum(0)
    place = count + back[-1] - 1 - ((back - freed)[:, None] + col - kept[:, None])
    mine = (col >= kept[:, None]) & (col < have[:, None])
    stack.scatter_(0, torch.where(mine, place, dump).reshape(-1), table.reshape(-1))
    top = count + back[-1]
    ends = n.cumsum(0)
    fits = ((keep + n) <= W * P) & (ends <= T)
    want = torch.where(fits, (keep + n + P - 1) // P - kept, 0)
    taken = want.cumsum(0)
    ok = fits & ((want == 0) | (taken <= top))
    want = torch.where(ok, want, 0)
    first = want.cumsum(0) - want
    place = top - 1 - (first[:, None] + col - kept[:, None])
    mine = (col >= kept[:, None]) & (col < (kept + want)[:, None])
    table.copy_(torch.where(mine, stack[torch.where(mine, place, dump)], table))
    free.copy_(stack[:N])
    count.copy_((top - want.sum()).to(torch.int32))
    s["lens"].copy_(torch.where(ok, keep + n, keep).to(torch.int32))
    starts = torch.cat([ends.new_zeros(1), ends]).clamp(max=T)
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    inside = r < R
    r = r.clamp(max=R - 1)
    pos = keep[r] + t - starts[r]
    inside &= ok[r]
    page = table[r, (pos // P).clamp(0, W - 1)].long()
    slots = torch.where(inside, page * P + pos % P, -1)
    return {"slots": slots, "starts": starts.to(torch.int32), "status": (~ok).to(torch.int32)}


def _scale_exponent(amax):
    """k of the least power of two 2^k that brings amax under e4m3's largest value, 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, (e - 9 + (m > 0.875)).clamp(min=SCALE_FLOOR), SCALE_FLOOR)


def _plain_store(x, slots, first, pages, scale, token_axis):
    """Writes the tokens x [T, H, D] of one of the two halves; `first`: the first token of each request."""
    P = pages.shape[token_axis]
    page, row = slots // P, slots % P
    x = x.float()
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    top = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand_as(amax), amax, "amax")
    lead, rows = page[first], row[first]                               # the only pages that hold older tokens
    old = torch.where(rows[:, None] > 0, scale[lead], 0.0)
    new = torch.ldexp(torch.ones_like(top), _scale_exponent(top))
    new[lead] = torch.maximum(new[lead], old)
    touched = torch.zeros_like(scale, dtype=torch.bool).index_fill_(0, page, True)
    live = torch.arange(P, device=DEV) < rows[:, None]
    live = live[:, None, :, None] if token_axis == 2 else live[:, None, None, :]
    was = pages[lead]
    again = was.float() * (old / new[lead])[..., None, None]
    pages[lead] = torch.where(live, again, was.float()).to(torch.float8_e4m3fn)
    scale.copy_(torch.where(touched, new, scale))
    stored = (x / new[page][..., None]).to(torch.float8_e4m3fn)
    if token_axis == 2:
        pages[page, :, row] = stored
    else:
        pages[page, :, :, row] = stored


def _plain_write(s):
    first = s["starts"][:-1].long()
    _plain_store(s["k"], s["slots"], first, s["k_pages"], s["k_scale"], 2)
    _plain_store(s["v"], s["slots"], first, s["v_pages"], s["v_scale"], 3)


def _plain_attend(s):
    case, table, lens = s["case"], s["table"].long().clamp(min=0), s["lens"].long()
    q = s["q"]
    T, Hq, D = q.shape
    R, W = table.shape
    Hkv, P = s["k_pages"].shape[1], case["P"]
    G, L = Hq // Hkv, W * P
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(R + 1, device=DEV)
    n = starts[1:] - starts[:-1]
    keys = torch.arange(L, device=DEV)
    held = keys < lens[:, None]
    k = (s["k_pages"][table].float() * s["k_scale"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(R, Hkv, L, D)
    v = (s["v_pages"][table].float() * s["v_scale"][table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(R, Hkv, L, D)
    v = torch.where(held[:, None, :, None], v, 0.0)
    i = torch.arange(s["most"], device=DEV)
    qp = q[(starts[:-1, None] + i).clamp(max=T - 1)].float()            # [R, most, Hq, D]
    qp = qp.reshape(R, -1, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hkv, -1, D)
    pos = lens[:, None] - n[:, None] + i                                # position of each query
    sees = held[:, None, :] & (keys <= pos[..., None])
    if case["window"]:
        sees &= keys > pos[..., None] - case["window"]
    x = torch.matmul(qp, k.transpose(2, 3).contiguous()).mul_(D ** -0.5).reshape(R, Hkv, G, -1, L)
    x = x.masked_fill_(~sees[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(m.isfinite(), m, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(R, Hkv, -1, L), v).reshape(R, Hkv, G, -1, D) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(R, -1, Hq, D)
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return o[r, t - starts[r]].to(q.dtype)


def _plain_sample(s):
    x = s["logits"].double()
    V = x.shape[1]
    x = torch.where(x.isnan(), -math.inf, x)
    temperature = s["temperature"].double()[:, None]
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((xs - xs[:, :1]) / temperature)
    rank = torch.arange(V, device=DEV)
    k = s["top_k"][:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    p = s["top_p"].double()[:, None]
    before = w.cumsum(1) - w
    w = torch.where((p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    c = w.cumsum(1)
    hit = (c > s["u"].double()[:, None] * c[:, -1:]) & (w > 0)
    return torch.where(hit.any(1), hit.int().argmax(1), -1)


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        from pigeon_amd import ops
    if op == "pages":
        if own:
            got = ops.page_advance(s["lens"], s["add"], s["table"], s["free"], s["count"], s["P"], s["T"], keep=s["keep"])
        else:
            got = _plain_pages(s)
        return {"slots": got["slots"], "starts": got["starts"], "status": got["status"], "lens": s["lens"], "table": s["table"],
                "free": s["free"], "count": s["count"]}
    if op == "write":
        if own:
            ops.cache_write(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
        else:
            _plain_write(s)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "attend":
        if own:
            return ops.cached_attention(s["q"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                                        starts=s["starts"], window=s["case"]["window"])
        return _plain_attend(s)
    if own:
        return ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return _plain_sample(s)


# ---------------------------------------------------------------------------------------------------- exact values
def _exact_pages(s):
    """Request by request, on a Python list as the stack of free pages."""
    P, T = s["P"], s["T"]
    lens, keep, add, table = (s[k].tolist() for k in ("lens", "keep", "add", "table"))
    count = s["count"].item()
    stack, rest = s["free"].tolist()[:count], s["free"].tolist()
    R, W = len(lens), len(table[0])
    back = [table[r][j] for r in range(R) for j in range(-(-keep[r] // P), -(-lens[r] // P))]
    stack += back[::-1]
    out = {"starts": [0], "status": [], "slots": np.full(T, -1, np.int64)}
    rest[:len(stack)] = stack
    end, full = 0, False
    for r in range(R):
        begin, end = end, end + add[r]
        out["starts"].append(min(end, T))
        have, want = -(-keep[r] // P), -(-(keep[r] + add[r]) // P)
        fits = keep[r] + add[r] <= W * P and end <= T
        full = full or (fits and want - have > len(stack))
        good = fits and (want == have or not full)
        out["status"].append(0 if good else 1)
        lens[r] = keep[r]
        if good:
            for j in range(have, want):
                table[r][j] = stack.pop()
            pos = keep[r] + np.arange(add[r])
            out["slots"][begin:end] = np.array(table[r], np.int64)[pos // P] * P + pos % P
            lens[r] += add[r]
    i32 = lambda v: np.array(v, np.int32)                                                                # noqa: E731
    return {"slots": out["slots"], "starts": i32(out["starts"]), "status": i32(out["status"]), "lens": i32(lens), "table": i32(table),
            "free": i32(rest), "count": i32([len(stack)])}


def _e4m3(x):
    """The nearest value of the 8-bit type (four significant bits, steps of 2^-9 at least, ties to even), in 64 bits."""
    e = np.maximum(np.frexp(x)[1] - 1, -6)
    step = np.ldexp(1.0, e - 3)
    return np.rint(x / step) * step


def _exact_store(x, slots, starts, pages, scale, P, token_axis):
    x, slots = x.double().cpu().numpy(), slots.cpu().numpy()
    held, scale = np.moveaxis(pages.double().cpu().numpy(), token_axis, 2), scale.double().cpu().numpy()     # [N, H, P, D]
    for a, b in zip(starts[:-1], starts[1:]):
        while a < b:
            page, row = divmod(int(slots[a]), P)
            c = min(b, a + P - row)
            new = np.moveaxis(x[a:c], 0, 1)                                   # [H, tokens, D]
            k = np.maximum(np.ceil(np.log2(np.maximum(np.abs(new).max((1, 2)) / 448, 2.0 ** SCALE_FLOOR))), SCALE_FLOOR)
            to = 2.0 ** k if row == 0 else np.maximum(2.0 ** k, scale[page])
            held[page, :, :row] = _e4m3(held[page, :, :row] * (scale[page] / to)[:, None, None])
            held[page, :, row:row + c - a] = _e4m3(new / to[:, None, None])
            scale[page] = to
            a = c
    return np.ascontiguousarray(np.moveaxis(held, 2, token_axis)), scale


def _exact_attend(s):
    case, P, D = s["case"], s["case"]["P"], s["case"]["D"]
    lens, new = _lengths(case)
    G = case["Hq"] // case["Hkv"]
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV), 0
    for r, (L, n) in enumerate(zip(lens, new)):
        page = s["table"][r, :-(-L // P)].long()
        key = torch.arange(L, device=DEV)
        pos = torch.arange(L - n, L, device=DEV)[:, None]
        off = key > pos
        if case["window"]:
            off |= key <= pos - case["window"]
        for h in range(case["Hkv"]):
            k = (s["k_pages"][page, h].double() * s["k_scale"][page, h].double()[:, None, None]).reshape(-1, D)[:L]
            v = (s["v_pages"][page, h].double() * s["v_scale"][page, h].double()[:, None, None]).transpose(1, 2).reshape(-1, D)[:L]
            q = s["q"][at:at + n, h * G:(h + 1) * G].double().transpose(0, 1).reshape(-1, D)
            x = (q @ k.T / math.sqrt(D)).reshape(G, n, L).masked_fill_(off, -math.inf)
            p = (x - x.amax(-1, keepdim=True)).exp_()
            p /= p.sum(-1, keepdim=True)
            out[at:at + n, h * G:(h + 1) * G] = (p.reshape(-1, L) @ v).reshape(G, n, D).transpose(0, 1)
        at += n
    return out


def _exact_sample(s):
    x, u, t, k, p, q = (s[n].double().cpu().numpy() for n in ("logits", "u", "temperature", "top_k", "top_p", "min_p"))
    ids = np.full(len(x), -1, np.int64)
    for b in range(len(x)):
        order = np.argsort(-x[b], kind="stable")
        order = order[:int(k[b])] if k[b] > 0 else order
        w = np.exp((x[b][order] - x[b].max()) / t[b])
        if p[b] < 1:
            keep = int(np.searchsorted(np.cumsum(w), p[b] * np.sum(w), side="left")) + 1
            order, w = order[:keep], w[:keep]
        order, w = order[w >= q[b]], w[w >= q[b]]
        by = np.argsort(order)
        c = np.cumsum(w[by])
        ids[b] = order[by][min(int(np.searchsorted(c, u[b] * c[-1], side="right")), len(c) - 1)]
    return ids


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return _exact_pages(s)
    if case["op"] == "write":
        if s["k_pages"].numel() > 1 << 27:
            return None
        starts = s["starts"].tolist()
        got = {}
        got["k_pages"], got["k_scale"] = _exact_store(s["k"], s["slots"], starts, s["k_pages"], s["k_scale"], case["P"], 2)
        got["v_pages"], got["v_scale"] = _exact_store(s["v"], s["slots"], starts, s["v_pages"], s["v_scale"], case["P"], 3)
        return got
    return _exact_attend(s) if case["op"] == "attend" else _exact_sample(s)
