"""The operators of the 4-bit cache as a list of cases: appending with the rotation on the way, reading rows back, attention
over the cache, attention over the pages that a cheap score selects.

``run`` makes the calls that a user makes of them where ``own`` is true, and computes the same by elementary torch
operations where it is false.  ``exact`` computes it in 64 bits by another route.

The cache: one record of 20 * D bytes per (page, kv head, 16 tokens), in 32-bit words (G = D / 32 groups of channels)

* ``8 D`` bytes of key codes: word ``(tau * 4 + t) * G + j`` holds channels ``32 j + 8 t + 0..7`` of token ``tau``;
* ``8 D`` bytes of value codes: word ``(32 h + 4 g + t) * G + j`` holds channels ``32 j + 4 g + 0..3`` of the tokens
  ``8 h + 2 t`` (low half) and ``8 h + 2 t + 1`` (high half);
* ``2 D`` bytes of key parameters, word ``tau * G + j`` = bf16 scale << 16 | bf16 zero, and ``2 D`` of value parameters.

A value is ``zero + scale * code``.  The summary holds each page's channel maxima and minima of the (rotated) keys.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LARGEST = 2.0 ** 126          # what the quantizer takes values to be at most
SMALLEST = 2.0 ** -96         # a smaller scale counts as none
# of a quotient that is then rounded: one that is a bf16 number stays that scale, one that lies between two codes goes to the
# lower one. 16-bit values meet both often, and by the quotient alone its last bit would say where they go.
SHRINK = 1 - 2.0 ** -20
CHUNK = 1 << 17               # (token, kv head) units of history that are made at a time


def _case(op, batch, lo, hi, kv_heads=8, q_heads=32, head_dim=128, page=16, dtype="bf16", **more):
    return {"op": op, "batch": batch, "len_lo": lo, "len_hi": hi, "kv_heads": kv_heads, "q_heads": q_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype, "new_lo": 0, "new_hi": 0, "pad": 0, "rot": 0, "interleaved": False, "budget": 0,
            "first": 0, "last": 0, "cap": 0.0, **more}


def listed():
    return [
        # a chat turn's token: one new row of one sequence, where latency is all
        {"name": "append_1", **_case("append", 1, 1000, 1000, new_lo=1, new_hi=1, rot=128)},
        # a served decode step: one new row of each of 61 ragged sequences, the batch padded to 64
        {"name": "append_step_61", **_case("append", 61, 17, 8191, kv_heads=8, q_heads=64, page=32, new_lo=1, new_hi=1, pad=3, rot=128)},
        # chunks of three prompts behind what is cached already, half of each head rotated, pairs side by side
        {"name": "append_chunks_3", **_case("append", 3, 1777, 4099, kv_heads=4, q_heads=16, dtype="f16", new_lo=333, new_hi=1025,
                                            rot=64, interleaved=True)},
        # a whole prompt of 8192 tokens
        {"name": "append_prompt_8k", **_case("append", 1, 8192, 8192, new_lo=8192, new_hi=8192, page=64, rot=128)},
        # the history of a chunked prefill's sequence, read back for the chunk's own attention
        {"name": "gather_b2_5k", **_case("gather", 2, 999, 5001)},
        {"name": "gather_64k_h64", **_case("gather", 1, 65536, 65536, head_dim=64, q_heads=32, dtype="f16", page=32)},
        # the first tokens of a chat: launches and latency
        {"name": "decode_333", **_case("decode", 1, 333, 333)},
        # a long document
        {"name": "decode_64k", **_case("decode", 1, 65536, 65536)},
        # a served batch of ragged lengths, eight query heads to a kv head
        {"name": "decode_b32_ragged", **_case("decode", 32, 700, 8191, q_heads=64, page=32, dtype="f16")},
        # the largest: eight long documents
        {"name": "decode_b8_64k", **_case("decode", 8, 65536, 65536)},
        # long documents of which a few percent are read
        {"name": "sparse_128k", **_case("sparse", 1, 131072, 131072, budget=256, first=1, last=4)},
        {"name": "sparse_b7_ragged", **_case("sparse", 7, 2049, 50021, kv_heads=4, q_heads=28, page=64, budget=33, first=1, last=2)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "gather", "decode", "decode", "sparse"))
    kv = rng.choice((1, 2, 3, 4, 8))
    D, page = rng.choice((64, 128, 128)), rng.choice((16, 16, 32, 64))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    q_heads = kv * rng.choice((1, 2, 4, 5, 7, 8))
    per_token = kv * D / 128
    if op == "append":
        new = _log(rng, 1, 8192)
        batch = max(1, min(_log(rng, 1, 64), 8192 // new))
        kept = _log(rng, 1, 8192)
        rot = rng.choice((32, 64, D))
        return _case(op, batch, new + kept // 3, new + kept, kv, q_heads, D, page, dtype, new_lo=max(1, new // 2), new_hi=new,
                     pad=rng.choice((0, 0, 5)), rot=rot, interleaved=rng.random() < 0.3)
    if op == "gather":
        batch = _log(rng, 1, 8)
        hi = _log(rng, 30, int(min(65536, 65536 * 4 / per_token / batch)))
        return _case(op, batch, max(1, hi // 3), hi, kv, q_heads, D, page, dtype)
    batch = _log(rng, 1, 64)
    hi = _log(rng, 20, int(min(131072, 65536 * 8 * 8 / per_token / batch)))
    if op == "decode":
        return _case(op, batch, max(1, hi // rng.choice((1, 3, 9))), hi, kv, q_heads, D, page, dtype, cap=rng.choice((0.0, 0.0, 0.0, 30.0)))
    budget = _log(rng, 4, 300)
    return _case(op, batch, max(1, hi // rng.choice((1, 3))), hi, kv, q_heads, D, page, dtype, budget=budget, first=1, last=min(budget - 1, 3))


# ---- shapes ----------------------------------------------------------------------------------------------------------
def _lens(c, lo, hi):
    return [c[hi] if i == 0 else c[lo] + int((c[hi] - c[lo]) * (i * 0.6180339887 % 1.0)) for i in range(c["batch"])]


def _shape(c):
    """Lengths, rows to append or read of each sequence, pages of each sequence."""
    lens = _lens(c, "len_lo", "len_hi")
    new = [min(n, m) for n, m in zip(_lens(c, "new_lo", "new_hi"), lens)] if c["op"] == "append" else list(lens)
    return lens, new, [-(-n // c["page"]) for n in lens]


def work(case):
    lens, new, pages = _shape(case)
    H, Hq, D = case["kv_heads"], case["q_heads"], case["head_dim"]
    unit = 20 * D / 16                                   # bytes of one token of one kv head
    table = 4 * sum(pages)
    if case["op"] == "append":                           # the rows and the query in, the record bytes and the query out, rows read back
        n = sum(new)
        touched = sum(-(-L // case["page"]) - (L - m) // case["page"] for L, m in zip(lens, new))
        return {"bytes": n * (2 * H + 2 * Hq) * D * 2 + 2 * n * H * unit + 2 * n * H * D * 2 + touched * H * 4 * D + n * case["rot"] * 4 + table,
                "flops": n * (2 * H * D * 10 + Hq * case["rot"] * 3)}
    if case["op"] == "gather":
        return {"bytes": sum(new) * H * (unit + 4 * D) + table, "flops": sum(new) * H * 4 * D}
    io = case["batch"] * Hq * (2 * D * 2 + 4)
    if case["op"] == "decode":
        return {"bytes": sum(lens) * H * unit + io + table, "flops": 4 * sum(lens) * Hq * D}
    read = sum(min(L, case["budget"] * case["page"]) for L in lens)
    return {"bytes": sum(pages) * H * 4 * D + read * H * unit + io + table + 8 * case["batch"] * H * case["budget"],
            "flops": 4 * read * Hq * D + 2 * sum(pages) * Hq * D}


# ---- the quantizer and the record, plain ------------------------------------------------------------------------------
def _floor_bf16(x):
    """Largest bf16 not above x (fp32 in, fp32 out)."""
    b = x.contiguous().view(torch.int32)
    cut = b & -65536
    return torch.where((b < 0) & (cut != b), cut + 65536, cut).view(torch.float32)


def _ceil_bf16(x):
    return -_floor_bf16(-x)


def _finite(x):
    return torch.nan_to_num(x.float(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST)


def _quantize(x):
    """x [..., D] -> codes [..., D] uint8, zero and scale [..., G] (fp32 values that bf16 holds)."""
    g = x.unflatten(-1, (-1, 32))
    zero = _floor_bf16(g.amin(-1))
    scale = _ceil_bf16((g.amax(-1) - zero) * (SHRINK / 15.0))
    scale = torch.where(scale < SMALLEST, torch.zeros_like(scale), scale)
    inverse = torch.where(scale > 0, SHRINK / scale, torch.zeros_like(scale))
    codes = ((g - zero[..., None]) * inverse[..., None]).round().clamp(0, 15)
    return codes.to(torch.uint8).flatten(-2), zero, scale


def _params(zero, scale):
    """[..., G] -> bytes [..., 4 G]"""
    return torch.stack((zero, scale), -1).to(torch.bfloat16).flatten(-2).view(torch.uint8)


def _nibbles(codes):
    """[..., 2 n] -> bytes [..., n], the even ones low."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _k_bytes(codes):
    """[..., D] of a token -> its D / 2 bytes: [t][j][8 channels]"""
    G = codes.shape[-1] // 32
    return _nibbles(codes.unflatten(-1, (G, 4, 8)).transpose(-3, -2).flatten(-3))


def _v_halves(codes):
    """[..., D] of a token -> its half words [..., g, j] (int16)"""
    G = codes.shape[-1] // 32
    return _nibbles(codes.unflatten(-1, (G, 8, 4)).transpose(-3, -2).contiguous()).view(torch.int16).squeeze(-1)


def _views(records):
    """Views of the four parts of records [P, H, S, 20 D] by token."""
    D = records.shape[-1] // 20
    G = D // 32
    kc = records[..., :8 * D].unflatten(-1, (16, D // 2))
    vc = records[..., 8 * D:16 * D].view(torch.int16).unflatten(-1, (2, 8, 4, G, 2))        # h, g, t, j, parity
    kp = records[..., 16 * D:18 * D].unflatten(-1, (16, 4 * G))
    vp = records[..., 18 * D:].unflatten(-1, (16, 4 * G))
    return kc, vc, kp, vp


def _pack(k, v):
    """k, v [N, 16, D] (values) -> records [N, 20 D]"""
    N, _, D = k.shape
    out = torch.empty(N, 20 * D, dtype=torch.uint8, device=k.device)
    kc, vc, kp, vp = _views(out)
    code, zero, scale = _quantize(k)
    kc.copy_(_k_bytes(code))
    kp.copy_(_params(zero, scale))
    code, zero, scale = _quantize(v)
    vc.copy_(_v_halves(code).unflatten(1, (2, 4, 2)).permute(0, 1, 4, 2, 5, 3))           # h, t, parity, g, j -> h, g, t, j, parity
    vp.copy_(_params(zero, scale))
    return out


def _unpack(records):
    """records [..., 20 D] -> keys and values [..., 16, D] in fp32"""
    D = records.shape[-1] // 20
    G = D // 32

    def spread(b):
        return torch.stack((b & 15, b >> 4), -1).flatten(-2)

    def values(code, par):
        p = par.contiguous().view(torch.bfloat16).unflatten(-1, (16, G, 2)).float()
        return (code.unflatten(-1, (G, 32)).float() * p[..., 1:2] + p[..., 0:1]).flatten(-2)

    kc = spread(records[..., :8 * D]).unflatten(-1, (16, 4, G, 8)).transpose(-3, -2).flatten(-3)
    vc = spread(records[..., 8 * D:16 * D]).unflatten(-1, (2, 8, 4, G, 2, 4))              # h, g, t, j, parity, i
    n = vc.dim() - 6
    vc = vc.permute(*range(n), n, n + 2, n + 4, n + 3, n + 1, n + 5).flatten(-3).flatten(-4, -2)
    return values(kc, records[..., 16 * D:18 * D]), values(vc, records[..., 18 * D:])


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens, new, pages = _shape(c)
    B, H, Hq, D, page, dt = c["batch"], c["kv_heads"], c["q_heads"], c["head_dim"], c["page"], DTYPES[c["dtype"]]
    P = sum(pages) + 3

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    # keys: channels of their own offset, a few of them large, pages that drift; values without either
    offset = rand(H, 1, D) * torch.where(torch.rand(H, 1, D, generator=gen, device=dev) < 0.05, 6.0, 0.5)
    records = torch.empty(P, H, page // 16, 20 * D, dtype=torch.uint8, device=dev)
    summary = torch.empty(P, H, 2, D, dtype=torch.bfloat16, device=dev)
    for p in range(0, P, max(1, CHUNK // (page * H))):
        n = min(max(1, CHUNK // (page * H)), P - p)
        k = (offset + 0.5 * rand(n, H, 1, D) + rand(n, H, page, D)).to(dt)
        records[p:p + n] = _pack(k.float().reshape(-1, 16, D), rand(n * H * page // 16, 16, D, dtype=dt).float()).view(n, H, page // 16, -1)
        summary[p:p + n, :, 0] = _ceil_bf16(k.float().amax(2)).to(torch.bfloat16)
        summary[p:p + n, :, 1] = _floor_bf16(k.float().amin(2)).to(torch.bfloat16)
    order = torch.randperm(P, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": c, "records": records, "summary": summary, "table": table, "max_len": max(lens),
         "b_seq_len": torch.tensor(lens, dtype=torch.int32, device=dev), "status": torch.zeros(1, dtype=torch.int32, device=dev)}
    if c["op"] in ("append", "gather"):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        T = starts[-1] + c["pad"]
        s["row_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        s["rows"] = starts[-1]
        s["k_out"], s["v_out"] = (torch.zeros(T, H, D, dtype=dt, device=dev) for _ in range(2))
        if c["op"] == "append":
            qkv = rand(T, Hq + 2 * H, D).to(dt)          # one projection's output, sliced
            qkv[:, Hq:Hq + H] += offset[:, 0].to(dt)
            s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
            s["q_out"] = torch.zeros(T, Hq, D, dtype=dt, device=dev)
            angle = torch.arange(max(lens), device=dev, dtype=torch.float64)[:, None] * \
                500000.0 ** (-torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s
    s["q"] = (rand(B, Hq, D) + 0.3 * offset.repeat_interleave(Hq // H, 0)[:, 0]).to(dt)
    s["o"] = torch.empty(B, Hq, D, dtype=dt, device=dev)
    s["lse"] = torch.empty(B, Hq, dtype=torch.float32, device=dev)
    if c["op"] == "sparse":
        s["selected"] = torch.empty(B, H, c["budget"], dtype=torch.int32, device=dev)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, interleaved):
    """x [T, heads, D] with the first 2 * cos.shape[-1] channels rotated, in x's type."""
    half = cos.shape[-1]
    f, c, s = x.float(), cos[:, None], sin[:, None]
    a, b = (f[..., 0:2 * half:2], f[..., 1:2 * half:2]) if interleaved else (f[..., :half], f[..., half:2 * half])
    y, z = a * c - b * s, b * c + a * s
    turned = torch.stack((y, z), -1).flatten(-2) if interleaved else torch.cat((y, z), -1)
    return torch.cat((turned, f[..., 2 * half:]), -1).to(x.dtype)


def _places(s):
    """Of every row: its position, page, 16-token part of the page and token of that."""
    n, page = s["rows"], s["case"]["page"]
    start = s["row_start"].long()
    seq = torch.searchsorted(start, torch.arange(n, device=start.device), right=True) - 1
    pos = s["b_seq_len"].long()[seq] - start[seq + 1] + torch.arange(n, device=start.device)
    return pos, s["table"][seq, pos // page].long(), pos % page // 16, pos % 16


def _append_plain(s):
    n = s["rows"]
    pos, page, part, tau = _places(s)
    cos, sin, turn = s["cos"][pos], s["sin"][pos], s["case"]["interleaved"]
    s["q_out"][:n] = _rotate(s["q"][:n], cos, sin, turn)
    k, v = _finite(_rotate(s["k"][:n], cos, sin, turn)), _finite(s["v"][:n])
    kc, vc, kp, vp = _views(s["records"])
    code, zero, scale = _quantize(k)
    kc[page, :, part, tau] = _k_bytes(code)
    kp[page, :, part, tau] = _params(zero, scale)
    code, zero, scale = _quantize(v)
    vc[page, :, part, tau // 8, :, tau % 8 // 2, :, tau % 2] = _v_halves(code)
    vp[page, :, part, tau] = _params(zero, scale)
    fresh = page[pos % s["case"]["page"] == 0]
    high, low = s["summary"][:, :, 0].float(), s["summary"][:, :, 1].float()
    high[fresh], low[fresh] = -math.inf, math.inf
    s["summary"][:, :, 0] = _ceil_bf16(high.index_reduce_(0, page, k, "amax"))
    s["summary"][:, :, 1] = _floor_bf16(low.index_reduce_(0, page, k, "amin"))
    _gather_plain(s)


def _gather_plain(s):
    n = s["rows"]
    _, page, part, tau = _places(s)
    kc, vc, kp, vp = _views(s["records"])
    G = kp.shape[-1] // 4

    def values(code, par):
        p = par.contiguous().view(torch.bfloat16).unflatten(-1, (G, 2)).float()
        return (code.float() * p[..., 1:2] + p[..., 0:1]).flatten(-2).to(s["k_out"].dtype)

    b = kc[page, :, part, tau].unflatten(-1, (4, G, 4))
    code = torch.stack((b & 15, b >> 4), -1).flatten(-2).transpose(-3, -2).flatten(-2)
    s["k_out"][:n] = values(code, kp[page, :, part, tau])
    b = vc[page, :, part, tau // 8, :, tau % 8 // 2, :, tau % 2].contiguous().view(torch.uint8).unflatten(-1, (G, 2))
    code = torch.stack((b & 15, b >> 4), -1).flatten(-2).transpose(-3, -2).flatten(-2)
    s["v_out"][:n] = values(code, vp[page, :, part, tau])


def _attend_plain(s, chosen, places):
    """chosen [B, H, n]: physical pages; places [B, H, n]: their places in the sequence, -1 for none."""
    c, q = s["case"], s["q"].float()
    B, Hq, D = q.shape
    H = c["kv_heads"]
    heads = torch.arange(H, device=q.device)[None, :, None]
    k, v = (x.flatten(2, 4) for x in _unpack(s["records"][chosen.long(), heads]))          # [B, H, tokens, D]
    token = places.long()[..., None] * c["page"] + torch.arange(c["page"], device=q.device)
    seen = ((places[..., None] >= 0) & (token < s["b_seq_len"].long()[:, None, None, None])).flatten(2)
    logit = (q.view(B, H, -1, D) @ k.transpose(-1, -2)) / math.sqrt(D)
    if c["cap"]:
        logit = c["cap"] * torch.tanh(logit / c["cap"])
    logit = logit.masked_fill(~seen[:, :, None], -math.inf)
    top = logit.amax(-1, keepdim=True)
    p = torch.exp(logit - top)
    total = p.sum(-1, keepdim=True)
    s["o"].copy_(((p @ v) / total).view(B, Hq, D))
    s["lse"].copy_((top + total.log()).view(B, Hq))


def _select_plain(s):
    c, q = s["case"], s["q"].float()
    B, Hq, D = q.shape
    H, n, P = c["kv_heads"], c["budget"], s["table"].shape[1]
    g = q.view(B, H, -1, D)
    _, e = torch.frexp(g.abs().amax((2, 3), keepdim=True))                                  # largest = m 2^e, m in [1/2, 1)
    qi = torch.ldexp(g, 7 - e).round().clamp(-127, 127)                                     # [B, H, heads, D]
    m = s["summary"][s["table"].long()].float().transpose(1, 2)                             # [B, H, P, 2, D]
    _, e = torch.frexp(m.abs().amax((3, 4)))
    e = (e - 1).clamp(min=-100)
    mi = (m * torch.ldexp(torch.full_like(m[:, :, :, 0, 0], 63 / 64), 5 - e)[..., None, None]).round()
    # whole numbers below 2^24: exact in 32 bits, in any order
    total = qi.clamp(min=0) @ mi[:, :, :, 0].transpose(-1, -2) + qi.clamp(max=0) @ mi[:, :, :, 1].transpose(-1, -2)
    key = total.amax(2).double() * torch.ldexp(torch.ones_like(e, dtype=torch.float64), e - 26)
    pages = (s["b_seq_len"].long() + c["page"] - 1) // c["page"]
    at, count = torch.arange(P, device=q.device), pages[:, None, None]
    key = key.masked_fill((at < c["first"]) | (at >= count - c["last"]), math.inf).masked_fill(at >= count, -math.inf)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :n]
    best = torch.where(best < count, best, P).sort(-1).values
    s["selected"].fill_(-1)
    s["selected"][..., :best.shape[-1]] = torch.where(best < count, best, -1)


def run(state):
    s, c = state, state["case"]
    if own:
        from open_ommx_serve_b200.attention.kv4 import (ommx_kv4_append, ommx_kv4_decode_attention, ommx_kv4_gather,
                                                        ommx_kv4_select_pages)
        if c["op"] == "append":
            ommx_kv4_append(s["k"], s["v"], s["records"], s["table"], s["b_seq_len"], row_start=s["row_start"], q=s["q"], q_out=s["q_out"],
                            cos=s["cos"], sin=s["sin"], interleaved=c["interleaved"], summary=s["summary"], status=s["status"])
        if c["op"] in ("append", "gather"):
            ommx_kv4_gather(s["records"], s["table"], s["b_seq_len"], s["k_out"], s["v_out"], row_start=s["row_start"], status=s["status"])
        if c["op"] == "sparse":
            ommx_kv4_select_pages(s["q"], s["summary"], s["table"], s["b_seq_len"], s["selected"], page_size=c["page"],
                                  first_pages=c["first"], last_pages=c["last"], status=s["status"])
        if c["op"] in ("decode", "sparse"):
            ommx_kv4_decode_attention(s["q"], s["records"], s["table"], s["b_seq_len"], s["o"], s["lse"], sm_scale=1 / math.sqrt(c["head_dim"]),
                                      logit_cap=c["cap"], selected=s.get("selected"), max_seq_len=s["max_len"], status=s["status"])
    elif c["op"] == "append":
        _append_plain(s)
    elif c["op"] == "gather":
        _gather_plain(s)
    elif c["op"] == "decode":
        places = torch.arange(s["table"].shape[1], device=s["table"].device).expand(c["batch"], c["kv_heads"], -1)
        _attend_plain(s, s["table"][:, None].expand(-1, c["kv_heads"], -1), places)
    else:
        _select_plain(s)
        chosen = s["table"].long()[:, None].expand(-1, c["kv_heads"], -1).gather(2, s["selected"].long().clamp(min=0))
        _attend_plain(s, chosen, s["selected"])
    if c["op"] == "append":
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"], "summary": s["summary"]}
    if c["op"] == "gather":
        return {"k": s["k_out"], "v": s["v_out"]}
    if c["op"] == "decode":
        return {"o": s["o"], "lse": s["lse"]}
    return {"selected": s["selected"], "o": s["o"], "lse": s["lse"]}


# ---- in 64 bits, by another route: byte by byte from the layout's formulas ----------------------------------------------
def _token64(rec, tokens, D):
    """rec [parts, 20 D] bytes of one (sequence, kv head), in order: keys and values [tokens, D] in 64 bits."""
    G, dev = D // 32, rec.device
    t = torch.arange(tokens, device=dev)[:, None]
    ch = torch.arange(D, device=dev)[None]
    flat, base, tau, j, r = rec.reshape(-1), t // 16 * (20 * D), t % 16, ch // 32, ch % 32

    def bf16_at(at):
        return ((flat[at].int() | flat[at + 1].int() << 8) << 16).view(torch.float32).double()

    def part(byte, nibble, par):
        code = (flat[byte].int() >> (4 * nibble)) & 15
        return bf16_at(par) + bf16_at(par + 2) * code

    word = (tau * 4 + r // 8) * G + j
    k = part(base + 4 * word + r % 8 // 2, (r % 2).expand_as(word), base + 16 * D + 4 * (tau * G + j))
    word = (tau // 8 * 32 + r // 4 * 4 + tau % 8 // 2) * G + j
    v = part(base + 8 * D + 4 * word + tau % 2 * 2 + r % 4 // 2, (r % 2).expand_as(word), base + 18 * D + 4 * (tau * G + j))
    return k, v


def _whole_bf16(x, up):
    """The bf16 number next above (or below) x, in 64 bits."""
    m, e = torch.frexp(x)
    return torch.ldexp((m * 256).ceil() if up else (m * 256).floor(), e - 8)


def _stored64(x):
    """What the cache holds of x [..., D]."""
    g = x.unflatten(-1, (-1, 32))
    low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    zero = _whole_bf16(low, False)
    step = _whole_bf16((high - zero) / 15 * SHRINK, True)
    step = torch.where(step < SMALLEST, 0.0, step)
    code = torch.where(step > 0, ((g - zero) / step.clamp(min=SMALLEST) * SHRINK).round().clamp(0, 15), 0.0)
    return (zero + step * code).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    c, (lens, new, _) = case, _shape(case)
    H, Hq, D, page = c["kv_heads"], c["q_heads"], c["head_dim"], c["page"]
    group = Hq // H
    if c["op"] == "append":
        q, k, v = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q_out", "k_out", "v_out"))
        summary = s["summary"].double()
        half, at = c["rot"] // 2, 0
        for b, (L, n) in enumerate(zip(lens, new)):
            angle = torch.complex(s["cos"][L - n:L].double(), s["sin"][L - n:L].double())[:, None]
            rows = slice(at, at + n)

            def turned(x):
                x = x[rows].double()
                z = x[..., :2 * half].unflatten(-1, (half, 2) if c["interleaved"] else (2, half))
                z = torch.complex(*z.unbind(-1 if c["interleaved"] else -2)) * angle
                z = torch.stack((z.real, z.imag), -1 if c["interleaved"] else -2).flatten(-2)
                return torch.cat((z, x[..., 2 * half:]), -1)

            q[rows] = turned(s["q"])
            key = turned(s["k"]).to(s["k"].dtype).double()
            k[rows], v[rows] = _stored64(key), _stored64(s["v"][rows].double())
            first, last = (L - n) // page, (L - 1) // page
            for p in range(first, last + 1):
                lo, hi = max(p * page, L - n), min((p + 1) * page, L)
                x, here = key[lo - (L - n):hi - (L - n)], int(s["table"][b, p])
                top, bottom = x.amax(0), x.amin(0)
                if lo > p * page:
                    top, bottom = torch.maximum(top, summary[here, :, 0]), torch.minimum(bottom, summary[here, :, 1])
                summary[here, :, 0], summary[here, :, 1] = _whole_bf16(top, True), _whole_bf16(bottom, False)
            at += n
        return {"q": q, "k": k, "v": v, "summary": summary}
    if c["op"] == "gather":
        k, v = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("k_out", "v_out"))
        at = 0
        for b, L in enumerate(lens):
            ids = s["table"][b, :-(-L // page)].long()
            for h in range(H):
                k[at:at + L, h], v[at:at + L, h] = _token64(s["records"][ids, h].flatten(0, 1), L, D)
            at += L
        return {"k": k, "v": v}
    o = torch.zeros(c["batch"], Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(c["batch"], Hq, dtype=torch.float64, device="cuda")
    selected = torch.full((c["batch"], H, max(1, c["budget"])), -1, dtype=torch.int32, device="cuda")
    for b, L in enumerate(lens):
        ids = s["table"][b, :-(-L // page)].long()
        for h in range(H):
            q = s["q"][b, h * group:(h + 1) * group].double()
            k, v = _token64(s["records"][ids, h].flatten(0, 1), L, D)
            if c["op"] == "sparse":
                top = int(math.floor(math.log2(float(q.abs().max()))))
                qi = (q * 2.0 ** (6 - top)).round().clamp(-127, 127)
                m = s["summary"][ids, h].double()
                e = torch.frexp(m.abs().flatten(1).max(1).values)[1].double() - 1
                mi = (m * (63 / 64) * torch.exp2(5 - e)[:, None, None]).round()
                score = torch.maximum(qi[:, None] * mi[None, :, 0], qi[:, None] * mi[None, :, 1]).sum(-1).max(0).values * torch.exp2(e)
                score[:c["first"]] = math.inf
                score[max(0, len(ids) - c["last"]):] = math.inf
                best = torch.sort(-score, stable=True).indices[:c["budget"]].sort().values
                selected[b, h, :len(best)] = best.int()
                token = (best[:, None] * page + torch.arange(page, device=best.device)).flatten()
                k, v = k[token[token < L]], v[token[token < L]]
            logit = q @ k.T / math.sqrt(D)
            if c["cap"]:
                logit = c["cap"] * torch.tanh(logit / c["cap"])
            o[b, h * group:(h + 1) * group] = torch.softmax(logit, -1) @ v
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(logit, -1)
    if c["op"] == "decode":
        return {"o": o, "lse": lse}
    return {"selected": selected, "o": o, "lse": lse}
