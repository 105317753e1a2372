"""The 4-bit cache restated word by word from its layout, and its operators in 64 bits.  Test infrastructure only."""
import math

import torch

LARGEST, SMALLEST, SHRINK = 2.0 ** 126, 2.0 ** -96, 1 - 2.0 ** -20


def to_bf16(x, up):
    """bf16 next above / below fp32 values, as fp32."""
    b = x.to(torch.bfloat16)
    wrong = (b.float() < x) if up else (b.float() > x)
    bits = b.view(torch.int16).int() & 0xFFFF
    away = (b.float() >= 0) == up                         # the magnitude grows towards the wanted side
    zero = (bits & 0x7FFF) == 0
    moved = torch.where(zero, torch.full_like(bits, 0x0001 if up else 0x8001), torch.where(away, bits + 1, bits - 1))
    bits = torch.where(wrong, moved, bits)
    return (bits << 16).view(torch.float32)


def finite(x):
    return torch.nan_to_num(x.float(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST)


def quantize(x):
    """x [..., D] in its own type -> codes [..., D], zero and scale [..., D / 32]; every step in fp32."""
    g = finite(x).unflatten(-1, (-1, 32))
    zero = to_bf16(g.min(-1).values + 0.0, up=False)
    scale = to_bf16((g.max(-1).values - zero) * torch.tensor(SHRINK / 15, dtype=torch.float32), up=True)
    scale = torch.where(scale < SMALLEST, torch.zeros_like(scale), scale)
    inverse = torch.where(scale > 0, torch.tensor(SHRINK, dtype=torch.float32) / scale, torch.zeros_like(scale))
    codes = torch.round((g - zero[..., None]) * inverse[..., None]).int().flatten(-2)
    assert int(codes.min()) >= 0 and int(codes.max()) <= 15
    return codes, zero, scale


def rotate(x, cos, sin, interleaved):
    """x [T, heads, D], cos / sin [T, rot / 2]: fp32, every product and sum rounded, then x's type."""
    half = cos.shape[-1]
    y = x.float().clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[:, None, i], sin[:, None, i]
        u, v = x[..., a].float(), x[..., b].float()
        y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    return y.to(x.dtype)


def put(records, page, head, part, tau, k, v):
    """Store a token's quantized key and value (k, v: (codes, zero, scale) of [D]) in records [P, H, S, 20 D] (uint8, CPU)."""
    D = records.shape[-1] // 20
    G = D // 32
    rec = records[page, head, part]
    words = rec.view(torch.int32)

    def bits(x):
        return int(x.reshape(1).to(torch.bfloat16).view(torch.int16).item()) & 0xFFFF

    def signed(w):
        return w - (1 << 32) if w >= 1 << 31 else w

    for j in range(G):
        for t in range(4):
            word = sum(int(k[0][32 * j + 8 * t + i]) << (4 * i) for i in range(8))
            words[(tau * 4 + t) * G + j] = signed(word)
        for g in range(8):
            half = sum(int(v[0][32 * j + 4 * g + i]) << (4 * i) for i in range(4))
            at = 2 * D + (32 * (tau // 8) + 4 * g + tau % 8 // 2) * G + j
            old = int(words[at]) & 0xFFFFFFFF
            words[at] = signed((old & 0x0000FFFF) | half << 16 if tau % 2 else (old & 0xFFFF0000) | half)
        words[4 * D + tau * G + j] = signed(bits(k[2][j]) << 16 | bits(k[1][j]))
        words[4 * D + D // 2 + tau * G + j] = signed(bits(v[2][j]) << 16 | bits(v[1][j]))


def values(records):
    """records [..., 20 D] uint8 -> K, V [..., 16, D] in 64 bits, by the layout's formulas."""
    D = records.shape[-1] // 20
    G = D // 32
    words = records.contiguous().view(torch.int32).long() & 0xFFFFFFFF
    tau, c = torch.arange(16)[:, None].to(records.device), torch.arange(D)[None].to(records.device)
    j = c // 32

    def real(w):
        return (w << 16).to(torch.int64).bitwise_and(0xFFFFFFFF).to(torch.int64)

    def f32(b):                                            # 32 bits as a float, in 64 bits
        b = torch.where(b >= 1 << 31, b - (1 << 32), b).to(torch.int32)
        return b.view(torch.float32).double()

    def part(word, shift, par):
        code = words[..., word] >> shift & 15
        w = words[..., par]
        return f32(real(w)) + f32(w & 0xFFFF0000) * code

    k = part((tau * 4 + c % 32 // 8) * G + j, 4 * (c % 8) + 0 * tau, 4 * D + tau * G + j)
    v = part(2 * D + (32 * (tau // 8) + 4 * (c % 32 // 4) + tau % 8 // 2) * G + j, 4 * (c % 4) + 16 * (tau % 2), 4 * D + D // 2 + tau * G + j)
    return k, v


def sequence(records, table, length):
    """K, V [H, length, D] in 64 bits of one sequence with page table row `table`."""
    P, H, S, _ = records.shape
    pages = -(-length // (16 * S))
    k, v = values(records[table[:pages].long().to(records.device)])          # [pages, H, S, 16, D]
    return tuple(x.transpose(0, 1).flatten(1, 3)[:, :length] for x in (k, v))


def attention(q, k, v, sm_scale, cap=0.0):
    """q [Hq, D], k / v [H, tokens, D] (or a list by kv head) in 64 bits -> o [Hq, D], lse [Hq]"""
    H = len(k)
    group = q.shape[0] // H
    o, lse = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    for h in range(q.shape[0]):
        kk, vv = k[h // group], v[h // group]
        if len(kk) == 0:
            continue
        x = kk @ q[h].double() * sm_scale
        if cap:
            x = cap * torch.tanh(x / cap)
        o[h], lse[h] = torch.softmax(x, 0) @ vv, torch.logsumexp(x, 0)
    return o, lse


def select(q, summary, table, length, page, n, first, last):
    """Pages of one sequence, by kv head: q [Hq, D], summary [P, H, 2, D] -> list of ascending lists.  Whole numbers of Python."""
    H, D = summary.shape[1], summary.shape[3]
    group = q.shape[0] // H
    pages = -(-length // page)
    out = []
    for h in range(H):
        if pages <= n:
            out.append(list(range(pages)))
            continue
        x = q[h * group:(h + 1) * group].double()
        top = float(x.abs().max())
        e = math.frexp(top)[1] - 1 if top else 0
        qi = torch.round(x * 2.0 ** (6 - e)).clamp(-127, 127).long()
        keys = []
        for p in range(pages):
            m = summary[int(table[p]), h].double()
            largest = float(m.abs().max())
            f = max(math.frexp(largest)[1] - 1 if largest else -127, -100)
            mi = torch.round(m * (63 / 64) * 2.0 ** (5 - f)).long()
            s = max(int(torch.maximum(qi[i] * mi[0], qi[i] * mi[1]).sum()) for i in range(group))
            keys.append(math.inf if p < first or p >= pages - last else math.ldexp(s, f))
        order = sorted(range(pages), key=lambda p: (-keys[p], p))
        out.append(sorted(order[:n]))
    return out
