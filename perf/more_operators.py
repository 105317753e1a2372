"""The operators of the 8-bit cache as a list of cases: appending rows, attention over the cache (whole, or the first tokens and a
sliding window), attention that keeps account of each token's weight, and eviction by that weight.

``run`` makes the calls that a user makes of them where ``own`` is true, and computes the same by elementary torch
operations where it is false.  ``exact`` computes it in 64 bits by another route.

The cache: ``codes`` [pages, kv heads, page / 16, 2, 16, D] in int8 or e4m3, keys and values of 16 tokens of a head (a block) one
after the other; ``scales`` uint8 [pages, kv heads, page / 16, 2], the exponents of their scales: a value is code * 2^(E - 127).
E is the smallest for which the block's largest value is at most 127 (int8) or 448 (e4m3) units, 0 for zeros alone; codes are rounded
to the nearest, ties to even.  A block that takes rows with a larger scale has the codes it holds rounded to that.
``weight`` fp32 [pages, kv heads, page]: what each token was attended to with.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
LARGEST = 2.0 ** 126          # what the quantizer takes values to be at most
CHUNK = 1 << 17               # (token, kv head) units of history that are made at a time


def _case(op, batch, lo, hi, kv_heads=8, q_heads=32, head_dim=128, page=16, dtype="bf16", codes="int8", **more):
    return {"op": op, "batch": batch, "len_lo": lo, "len_hi": hi, "kv_heads": kv_heads, "q_heads": q_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype, "codes": codes, "new_lo": 0, "new_hi": 0, "pad": 0, "cap": 0.0, "window": 0, "sinks": 0,
            "keep": 1.0, "budget": 0, "recent": 0, **more}


def listed():
    return [
        # a chat turn's token: one new row of one sequence, where latency is all; its block is read back
        {"name": "append_1", **_case("append", 1, 1000, 1000, new_lo=1, new_hi=1)},
        # a served decode step: one new row of each of 61 ragged sequences, the batch padded to 64
        {"name": "append_step_61", **_case("append", 61, 17, 8191, q_heads=64, page=32, codes="e4m3", new_lo=1, new_hi=1, pad=3)},
        # chunks of three prompts behind what is cached already
        {"name": "append_chunks_3", **_case("append", 3, 1777, 4099, kv_heads=4, q_heads=16, dtype="f16", new_lo=333, new_hi=1025)},
        # a whole prompt of 8192 tokens
        {"name": "append_prompt_8k", **_case("append", 1, 8192, 8192, new_lo=8192, new_hi=8192, page=64)},
        # the first tokens of a chat: launches and latency
        {"name": "decode_333", **_case("decode", 1, 333, 333)},
        # a served batch of ragged lengths, eight query heads to a kv head
        {"name": "decode_b32_ragged", **_case("decode", 32, 700, 8191, q_heads=64, page=32, dtype="f16", codes="e4m3")},
        # the largest: eight long documents
        {"name": "decode_b8_64k", **_case("decode", 8, 65536, 65536)},
        # a long chat of which the last 4096 tokens and the first four stay visible
        {"name": "window_128k", **_case("decode", 1, 131072, 131072, window=4096, sinks=4)},
        # a served batch with a window, some sequences shorter than it
        {"name": "window_b61_ragged", **_case("decode", 61, 300, 20011, q_heads=64, page=32, codes="e4m3", window=1025, sinks=17)},
        # a step over a long document that keeps account of what is attended to, for the eviction to come
        {"name": "weigh_64k", **_case("decode", 1, 65536, 65536, keep=0.999, weigh=True)},
        # the eviction: a long document down to 4096 tokens, its first and its last ones among them
        {"name": "evict_64k", **_case("evict", 1, 65536, 65536, budget=4096, sinks=4, recent=512)},
        # a served batch, some sequences shorter than what they may keep
        {"name": "evict_b16_ragged", **_case("evict", 16, 900, 9001, kv_heads=4, q_heads=28, page=64, codes="e4m3", dtype="f16",
                                             budget=1999, sinks=1, recent=256)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "decode", "decode", "window", "weigh", "evict"))
    kv = rng.choice((1, 2, 3, 4, 8))
    D, page = rng.choice((64, 128, 128)), rng.choice((16, 16, 32, 64))
    dtype, codes = rng.choice(("bf16", "bf16", "f16")), rng.choice(("int8", "e4m3"))
    q_heads = kv * rng.choice((1, 2, 4, 5, 7, 8, 16))
    per_token = kv * D / 128
    if op == "append":
        new = _log(rng, 1, 8192)
        batch = max(1, min(_log(rng, 1, 64), 8192 // new))
        kept = _log(rng, 1, 8192)
        return _case(op, batch, new + kept // 3, new + kept, kv, q_heads, D, page, dtype, codes, new_lo=max(1, new // 2), new_hi=new,
                     pad=rng.choice((0, 0, 5)))
    batch = _log(rng, 1, 64)
    hi = _log(rng, 20, int(min(131072, 65536 * 8 * 8 / per_token / batch / (2 if q_heads > 8 * kv else 1))))
    lo = max(1, hi // rng.choice((1, 3, 9)))
    if op == "evict":
        budget = _log(rng, min(hi, 20), min(hi, 8192) if batch < 9 else min(hi, 2048))
        return _case(op, batch, lo, hi, kv, q_heads, D, page, dtype, codes, budget=budget, sinks=rng.choice((0, 1, 4)) if budget > 4 else 0,
                     recent=budget // rng.choice((3, 5, 40)))
    more = {"cap": rng.choice((0.0, 0.0, 0.0, 30.0))}
    if op == "window":
        more.update(window=_log(rng, 1, hi), sinks=rng.choice((0, 1, 4, 17, 64)))
    if op == "weigh":
        more.update(weigh=True, keep=rng.choice((0.0, 0.9, 1.0)), window=rng.choice((0, 0, 333)), sinks=4)
    return _case("decode", batch, lo, hi, kv, q_heads, D, page, dtype, codes, **more)


# ---- shapes ----------------------------------------------------------------------------------------------------------
def _lens(c, lo, hi):
    return [c[hi] if i == 0 else c[lo] + int((c[hi] - c[lo]) * (i * 0.6180339887 % 1.0)) for i in range(c["batch"])]


def _shape(c):
    """Lengths, rows to append of each sequence, pages of each sequence, tokens that each keeps."""
    lens = _lens(c, "len_lo", "len_hi")
    new = [min(n, m) for n, m in zip(_lens(c, "new_lo", "new_hi"), lens)]
    return lens, new, [-(-n // c["page"]) for n in lens], [min(n, c["budget"]) for n in lens]


def _seen(c, n):
    return n if not c["window"] else min(n, c["window"] + c["sinks"])


def work(case):
    c, (lens, new, pages, kept) = case, _shape(case)
    H, Hq, D = c["kv_heads"], c["q_heads"], c["head_dim"]
    unit = 2 * D + 2 / 16                                # bytes of one token of one kv head
    table = 4 * sum(pages)
    if c["op"] == "append":                              # rows in, codes out; the blocks that they lie in read back
        back = sum(m + (L - m) % 16 for L, m in zip(lens, new))
        n = sum(new)
        return {"bytes": n * H * (4 * D + unit) + back * H * (unit + 4 * D) + table, "flops": (n + back) * H * 4 * D}
    if c["op"] == "evict":                               # all weights, the kept tokens in and out, and those read back
        n = sum(kept)
        return {"bytes": 4 * sum(lens) * H + n * H * (2 * unit + 12 + unit + 4 * D) + table, "flops": 4 * sum(lens) * H + n * H * 8 * D}
    seen = sum(_seen(c, n) for n in lens)
    io = c["batch"] * Hq * (2 * D * 2 + 4) + (8 * sum(lens) * H if c.get("weigh") else 0)
    return {"bytes": seen * H * unit + io + table, "flops": 4 * seen * Hq * D}


# ---- the quantizer, plain --------------------------------------------------------------------------------------------
def _finite(x):
    return torch.nan_to_num(x.float(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST)


def _exponent(top, codes):
    """E of a largest value (fp32): the smallest from 1 on with top <= TOP 2^(E - 127); 0 for none."""
    m, e = torch.frexp(top)                              # top = m 2^e, m in [1/2, 1)
    unit, shift = math.frexp(TOP[codes])
    e = e - shift + (m > unit).to(e.dtype) + 127
    return torch.where(top > 0, e.clamp(min=1), torch.zeros_like(e))


def _power(e):
    """2^e in fp32, e up to 127; 0 below -126"""
    return ((e.to(torch.int32) + 127).clamp(min=0) << 23).view(torch.float32)


def _codes(x, codes):
    """What x (fp32, in units) is held as."""
    return x.round().to(torch.int8) if codes == "int8" else x.to(torch.float8_e4m3fn)


def _quantize(x, codes):
    """x [..., 16, D] (fp32) -> codes and E [...]"""
    E = _exponent(x.abs().amax((-2, -1)), codes)
    return _codes(x * _power(127 - E.clamp(min=1))[..., None, None], codes), E.to(torch.uint8)


def _values(codes, E):
    """codes [..., 16, D], E [...] -> fp32"""
    return codes.float() * _power(E.int().clamp(min=1) - 127)[..., None, None]


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens, new, pages, kept = _shape(c)
    B, H, Hq, D, page, dt = c["batch"], c["kv_heads"], c["q_heads"], c["head_dim"], c["page"], DTYPES[c["dtype"]]
    room = [-(-n // page) for n in kept]                 # pages that take what is kept
    P = sum(pages) + sum(room) + 3

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    # keys: channels of their own offset, a few of them large, pages that drift; values of sizes that differ from page to page
    offset = rand(H, 1, D) * torch.where(torch.rand(H, 1, D, generator=gen, device=dev) < 0.05, 6.0, 0.5)
    codes = torch.empty(P, H, page // 16, 2, 16, D, dtype=CODES[c["codes"]], device=dev)
    scales = torch.empty(P, H, page // 16, 2, dtype=torch.uint8, device=dev)
    for p in range(0, P, max(1, CHUNK // (page * H))):
        n = min(max(1, CHUNK // (page * H)), P - p)
        k = offset + 0.5 * rand(n, H, 1, D) + rand(n, H, page, D)
        v = rand(n, H, page, D) * torch.exp(0.5 * rand(n, H, 1, 1))
        kv = torch.stack((k.unflatten(2, (-1, 16)), v.unflatten(2, (-1, 16))), 3).to(dt).float()
        held, E = _quantize(kv, c["codes"])
        codes[p:p + n].copy_(held)
        scales[p:p + n] = E
    order = torch.randperm(P, generator=gen, device=dev).to(torch.int32)
    table, to_table = torch.zeros(B, max(pages), dtype=torch.int32, device=dev), torch.zeros(B, max(room + [1]), dtype=torch.int32, device=dev)
    at = 0
    for t, counts in ((table, pages), (to_table, room)):
        for b, n in enumerate(counts):
            t[b, :n] = order[at:at + n]
            at += n
    s = {"case": c, "codes": codes, "scales": scales, "table": table, "max_len": max(lens),
         "b_seq_len": torch.tensor(lens, dtype=torch.int32, device=dev), "status": torch.zeros(1, dtype=torch.int32, device=dev)}

    def starts(counts):
        return torch.tensor([0] + counts, dtype=torch.int32, device=dev).cumsum(0).to(torch.int32)

    if c["op"] == "append":
        s["row_start"], s["rows"] = starts(new), sum(new)
        back = [m + (L - m) % 16 for L, m in zip(lens, new)]   # from the first token of the first block that is touched
        s["back_start"], s["back"] = starts(back), sum(back)
        T = s["rows"] + c["pad"]
        qkv = rand(T, Hq + 2 * H, D)                     # one projection's output, sliced
        qkv[:, Hq:Hq + H] += offset[:, 0]
        qkv = (qkv * torch.exp(0.5 * rand(T, 1, 1))).to(dt)
        s["k"], s["v"] = qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
        s["k_out"], s["v_out"] = (torch.zeros(s["back"], H, D, dtype=dt, device=dev) for _ in range(2))
        return s
    if c["op"] == "evict":
        # what accumulated: a few tokens hold most, many hold the same little, some were never looked at
        w = torch.exp(2.5 * rand(P, H, page))
        s["weight"] = torch.where(w < 0.2, 0.0, torch.where(w < 0.5, 0.25, w))
        s["to_table"], s["kept"] = to_table, torch.empty(B, H, c["budget"], dtype=torch.int32, device=dev)
        s["len_out"] = torch.zeros(B, dtype=torch.int32, device=dev)
        s["back_start"], s["back"] = starts(kept), sum(kept)
        s["k_out"], s["v_out"] = (torch.zeros(s["back"], H, D, dtype=dt, device=dev) for _ in range(2))
        return s
    s["q"] = (rand(B, Hq, D) + 0.3 * offset.repeat_interleave(Hq // H, 0)[:, 0]).to(dt)
    s["o"] = torch.empty(B, Hq, D, dtype=dt, device=dev)
    s["lse"] = torch.empty(B, Hq, dtype=torch.float32, device=dev)
    if c.get("weigh"):
        s["weight_before"] = torch.rand(P, H, page, generator=gen, device=dev) ** 8
        s["weight"] = torch.zeros(P, H, page, device=dev)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _places(s, table, start, length, n):
    """Of every row: its position, page, 16-token part of the page and token of that."""
    page = s["case"]["page"]
    start = start.long()
    seq = torch.searchsorted(start, torch.arange(n, device=start.device), right=True) - 1
    pos = length.long()[seq] - start[seq + 1] + torch.arange(n, device=start.device)
    return pos, table[seq, pos // page].long(), pos % page // 16, pos % 16


def _append_plain(s):
    c, n = s["case"], s["rows"]
    pos, page, part, tau = _places(s, s["table"], s["row_start"], s["b_seq_len"], n)
    kind = c["codes"]
    x = _finite(torch.stack((s["k"][:n], s["v"][:n]), 2))                                   # [rows, H, 2, D]
    block, of = torch.unique(page * (c["page"] // 16) + part, return_inverse=True)
    p, r = block // (c["page"] // 16), block % (c["page"] // 16)
    top = torch.zeros(len(block), *x.shape[1:3], device=x.device).index_reduce_(0, of, x.abs().amax(-1), "amax")
    first = torch.full((len(block),), 16, device=x.device).index_reduce_(0, of, tau, "amin")
    held = torch.where((first > 0)[:, None, None], s["scales"][p, :, r].int(), 0)
    E = torch.maximum(_exponent(top, kind), held)
    bytes_ = s["codes"].view(torch.uint8)
    old = bytes_[p, :, r].view(CODES[kind]).float()                                          # [blocks, H, 2, 16, D]
    old = _codes(old * _power(held - E).masked_fill(held == 0, 0.0)[..., None, None], kind).view(torch.uint8)
    bytes_[p, :, r] = torch.where((E > held)[..., None, None], old, bytes_[p, :, r])
    s["scales"][p, :, r] = E.to(torch.uint8)
    bytes_[page, :, part, :, tau] = _codes(x * _power(127 - E[of].clamp(min=1))[..., None], kind).view(torch.uint8)
    _gather_plain(s, s["table"], s["b_seq_len"])


def _gather_plain(s, table, length):
    _, page, part, tau = _places(s, table, s["back_start"], length, s["back"])
    held = s["codes"].view(torch.uint8)[page, :, part, :, tau].view(s["codes"].dtype).float()              # [rows, H, 2, D]
    x = held * _power(s["scales"][page, :, part].int().clamp(min=1) - 127)[..., None]
    s["k_out"].copy_(x[:, :, 0])
    s["v_out"].copy_(x[:, :, 1])


def _attend_plain(s):
    c, q = s["case"], s["q"].float()
    B, Hq, D = q.shape
    H, table = c["kv_heads"], s["table"].long()
    kv = s["codes"].view(torch.uint8)[table].view(s["codes"].dtype).float() * _power(s["scales"][table].int().clamp(min=1) - 127)[..., None, None]
    k, v = (kv[:, :, :, :, i].transpose(1, 2).flatten(2, 4) for i in range(2))               # [B, H, tokens, D]
    token, n = torch.arange(k.shape[2], device=q.device), s["b_seq_len"].long()[:, None]
    there = token < n
    seen = there & ((token < c["sinks"]) | (token >= n - c["window"])) if c["window"] else there
    logit = (q.view(B, H, -1, D) @ k.transpose(-1, -2)) / math.sqrt(D)
    if c["cap"]:
        logit = c["cap"] * torch.tanh(logit / c["cap"])
    logit = logit.masked_fill(~seen[:, None, None], -math.inf)
    top = logit.amax(-1, keepdim=True)
    p = torch.exp(logit - top)
    total = p.sum(-1, keepdim=True)
    s["o"].copy_(((p @ v) / total).view(B, Hq, D))
    s["lse"].copy_((top + total.log()).view(B, Hq))
    if c.get("weigh"):
        of, at = torch.nonzero(there, as_tuple=True)
        page, tau = table[of, at // c["page"]], at % c["page"]
        s["weight"][page, :, tau] = c["keep"] * s["weight_before"][page, :, tau] + (p / total).sum(2)[of, :, at]


def _evict_plain(s):
    c = s["case"]
    B, H, n, page = c["batch"], c["kv_heads"], c["budget"], c["page"]
    table, length = s["table"].long(), s["b_seq_len"].long()[:, None, None]
    w = s["weight"][table].transpose(1, 2).flatten(2)                                        # [B, H, tokens]
    at = torch.arange(w.shape[2], device=w.device)
    key = w.masked_fill((at < c["sinks"]) | (at >= length - c["recent"]), math.inf).masked_fill(at >= length, -math.inf)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :n]
    best = torch.where(best < length, best, w.shape[2]).sort(-1).values
    s["kept"].fill_(-1)
    s["kept"][..., :best.shape[-1]] = torch.where(best < length, best, -1)
    s["len_out"].copy_(length.view(B).clamp(max=n))
    # every place that takes a token: where it comes from, and the scale of the block that it is in
    seq, place = torch.nonzero(torch.arange(n, device=w.device) < length[:, 0], as_tuple=True)
    src, heads = s["kept"][seq, :, place].long(), torch.arange(H, device=w.device)            # [rows, H]
    from_page = table[seq[:, None], src // page]
    bytes_, kind = s["codes"].view(torch.uint8), c["codes"]
    code = bytes_[from_page, heads, src % page // 16, :, src % 16].view(CODES[kind]).float()  # [rows, H, 2, D]
    E = s["scales"][from_page, heads, src % page // 16].int()                                 # [rows, H, 2]
    weight = s["weight"][from_page, heads, src % page]
    block, of = torch.unique(seq * (n // 16 + 1) + place // 16, return_inverse=True)
    to = torch.zeros(len(block), H, 2, dtype=torch.int32, device=w.device).index_reduce_(0, of, E, "amax")[of]
    to_page, part, tau = s["to_table"].long()[seq, place // page], place % page // 16, place % 16
    code = code * _power(E - to).masked_fill(E == 0, 0.0)[..., None]
    bytes_[to_page, :, part, :, tau] = _codes(code, kind).view(torch.uint8)
    s["scales"][to_page, :, part] = to.to(torch.uint8)
    s["weight"][to_page, :, place % page] = weight
    _gather_plain(s, s["to_table"], s["len_out"])


def run(state):
    s, c = state, state["case"]
    if own:
        from open_ommx_serve_b200.attention.kv8 import ommx_kv8_append, ommx_kv8_decode_attention, ommx_kv8_evict, ommx_kv8_gather
        if c["op"] == "append":
            ommx_kv8_append(s["k"], s["v"], s["codes"], s["scales"], s["table"], s["b_seq_len"], row_start=s["row_start"], status=s["status"])
            ommx_kv8_gather(s["codes"], s["scales"], s["table"], s["b_seq_len"], s["k_out"], s["v_out"], row_start=s["back_start"],
                            status=s["status"])
        elif c["op"] == "evict":
            ommx_kv8_evict(s["codes"], s["scales"], s["weight"], s["table"], s["b_seq_len"], s["kept"], sink_tokens=c["sinks"],
                           recent_tokens=c["recent"], to_table=s["to_table"], len_out=s["len_out"], max_seq_len=s["max_len"], status=s["status"])
            ommx_kv8_gather(s["codes"], s["scales"], s["to_table"], s["len_out"], s["k_out"], s["v_out"], row_start=s["back_start"],
                            status=s["status"])
        else:
            ommx_kv8_decode_attention(s["q"], s["codes"], s["scales"], s["table"], s["b_seq_len"], s["o"], s["lse"],
                                      sm_scale=1 / math.sqrt(c["head_dim"]), logit_cap=c["cap"], window=c["window"] or None,
                                      sink_tokens=c["sinks"], weight=s.get("weight"), weight_before=s.get("weight_before"), keep=c["keep"],
                                      max_seq_len=s["max_len"], status=s["status"])
    elif c["op"] == "append":
        _append_plain(s)
    elif c["op"] == "evict":
        _evict_plain(s)
    else:
        _attend_plain(s)
    if c["op"] == "append":
        return {"k": s["k_out"], "v": s["v_out"]}
    if c["op"] == "evict":
        return {"kept": s["kept"], "len": s["len_out"], "k": s["k_out"], "v": s["v_out"], "weight": s["weight"]}
    return {"o": s["o"], "lse": s["lse"], **({"weight": s["weight"]} if c.get("weigh") else {})}


# ---- in 64 bits, by another route ---------------------------------------------------------------------------------------
def _power64(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _rounded64(x, codes):
    """x (in units) to the nearest code, ties to even"""
    if codes == "int8":
        return torch.round(x)
    step = _power64(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)                        # three bits behind the leading one
    return torch.round(x / step) * step


def _unit64(top, codes):
    """The power of two that a block of this largest value is held in; 0 for none."""
    low = _power64(torch.frexp(top / TOP[codes])[1].clamp(min=-125) - 1)                     # at most what is looked for
    return torch.where(top > 0, torch.where(top > low * TOP[codes], 2 * low, low), 0.0)


def _held64(s, ids, h):
    """Units [blocks, 2] and values [blocks, 2, 16, D] of one kv head's blocks of these pages, in order."""
    E = s["scales"][ids, h].flatten(0, 1).double()
    unit = torch.where(E > 0, _power64(E - 127), 0.0)
    return unit, s["codes"].view(torch.uint8)[ids, h].view(s["codes"].dtype).to(torch.float32).double().flatten(0, 1) * unit[..., None, None]


def exact(case, seed):
    s = prepare(case, seed)
    c, (lens, new, _, kept) = case, _shape(case)
    H, Hq, D, page, kind = c["kv_heads"], c["q_heads"], c["head_dim"], c["page"], c["codes"]
    group = Hq // H
    dev = s["codes"].device
    if c["op"] in ("append", "evict"):
        k, v = (torch.zeros(s["back"], H, D, dtype=torch.float64, device=dev) for _ in range(2))
    if c["op"] == "append":
        at = back = 0
        for b, (L, n) in enumerate(zip(lens, new)):
            ids = s["table"][b, :-(-L // page)].long()
            old, lead = L - n, (L - n) % 16
            for h in range(H):
                unit, held = _held64(s, ids, h)
                unit, held = unit[old // 16:-(-L // 16)].clone(), held[old // 16:-(-L // 16)]
                x = torch.zeros(len(unit) * 16, 2, D, dtype=torch.float64, device=dev)
                x[lead:lead + n, 0], x[lead:lead + n, 1] = s["k"][at:at + n, h].double(), s["v"][at:at + n, h].double()
                x = x.view(-1, 16, 2, D).transpose(1, 2)
                unit[1 if lead else 0:] = 0.0            # only the first block held tokens before
                now = torch.maximum(unit, _unit64(x.abs().amax((2, 3)), kind))
                x[0, :, :lead] = held[0, :, :lead] * (unit[0] > 0)[:, None, None]
                now = now[..., None, None]
                x = torch.where(now > 0, _rounded64(x / now.clamp(min=2.0 ** -126), kind) * now, 0.0).transpose(1, 2).flatten(0, 1)
                k[back:back + n + lead, h], v[back:back + n + lead, h] = x[:n + lead, 0], x[:n + lead, 1]
            at, back = at + n, back + n + lead
        return {"k": k, "v": v}
    if c["op"] == "evict":
        chosen = torch.full(s["kept"].shape, -1, dtype=torch.int32, device=dev)
        weight, at = s["weight"].double(), 0
        before = s["weight"].double()
        for b, (L, n) in enumerate(zip(lens, kept)):
            ids, to = s["table"][b, :-(-L // page)].long(), s["to_table"][b].long()
            for h in range(H):
                w = before[ids, h].flatten()[:L]
                score = w.clone()
                score[:c["sinks"]] = math.inf
                score[max(0, L - c["recent"]):] = math.inf
                best = torch.sort(-score, stable=True).indices[:n].sort().values
                chosen[b, h, :n] = best.int()
                place = torch.arange(n, device=dev)
                weight[to[place // page], h, place % page] = w[best]
                unit, held = _held64(s, ids, h)
                unit, x = unit[best // 16], held[best // 16, :, best % 16]                   # [n, 2], [n, 2, D]
                pad = torch.zeros(-n % 16, 2, dtype=torch.float64, device=dev)
                now = torch.cat((unit, pad)).view(-1, 16, 2).amax(1).repeat_interleave(16, 0)[:n, :, None]
                x = torch.where(now > 0, _rounded64(x / now.clamp(min=2.0 ** -126), kind) * now, 0.0)
                k[at:at + n, h], v[at:at + n, h] = x[:, 0], x[:, 1]
            at += n
        return {"kept": chosen, "len": torch.tensor(kept, dtype=torch.int32, device=dev), "k": k, "v": v, "weight": weight}
    o = torch.zeros(c["batch"], Hq, D, dtype=torch.float64, device=dev)
    lse = torch.zeros(c["batch"], Hq, dtype=torch.float64, device=dev)
    weight = s["weight"].double() if c.get("weigh") else None
    for b, L in enumerate(lens):
        ids = s["table"][b, :-(-L // page)].long()
        token = torch.arange(L, device=dev)
        if c["window"]:
            token = token[(token < c["sinks"]) | (token >= L - c["window"])]
        for h in range(H):
            held = _held64(s, ids, h)[1]
            x = held[token // 16, :, token % 16]
            logit = s["q"][b, h * group:(h + 1) * group].double() @ x[:, 0].T / math.sqrt(D)
            if c["cap"]:
                logit = c["cap"] * torch.tanh(logit / c["cap"])
            p = torch.softmax(logit, -1)
            o[b, h * group:(h + 1) * group] = p @ x[:, 1]
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(logit, -1)
            if c.get("weigh"):
                every = torch.arange(L, device=dev)
                now = c["keep"] * s["weight_before"][ids[every // page], h, every % page].double()
                now[token] += p.sum(0)
                weight[ids[every // page], h, every % page] = now
    return {"o": o, "lse": lse, **({"weight": weight} if c.get("weigh") else {})}
