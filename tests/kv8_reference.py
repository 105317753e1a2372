"""The 8-bit cache restated token by token, and its operators in 64 bits.  Test infrastructure only."""
import math

import torch

TOP = {torch.int8: 127, torch.float8_e4m3fn: 448}
LARGEST = 2.0 ** 126


def finite(x):
    return torch.nan_to_num(x.double(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST)


def exponent(top, dtype):
    """E of a largest value: the first from 1 on that holds it."""
    if top == 0:
        return 0
    E = max(1, math.frexp(top)[1] + 127 - 10)
    while top > TOP[dtype] * 2.0 ** (E - 127):
        E += 1
    return E


def rounded(x, dtype):
    """The nearest code of x (64 bits, in units), ties to even, as a number."""
    if dtype == torch.int8:
        return torch.round(x)
    out = torch.empty_like(x)
    for i, v in enumerate(x.flatten().tolist()):
        step = 2.0 ** (max(math.frexp(v)[1] - 1, -6) - 3)
        out.view(-1)[i] = math.copysign(round(v / step) * step, v)        # Python rounds ties to even; zeros keep their sign
    return out


def numbers(codes):
    return codes.to(torch.float32).double()


def as_codes(x, dtype):
    return x.to(torch.float32).to(dtype)                 # exact: x is a code's number


def append(codes, scales, weight, table, lens, starts, k, v):
    """Rows into a cache on the CPU, in place: a block at a time."""
    _, H, S, _, _, D = codes.shape
    page = 16 * S
    for b, L in enumerate(lens):
        n = starts[b + 1] - starts[b]
        for block in sorted({t // 16 for t in range(L - n, L)}):
            places = [t for t in range(L - n, L) if t // 16 == block]
            rows = [starts[b] + t - (L - n) for t in places]
            p, s, lead = int(table[b][block * 16 // page]), block % S, places[0] % 16
            for h in range(H):
                if weight is not None:
                    for t in places:
                        weight[p, h, t % page] = 0.0
                for i, x in enumerate((k, v)):
                    new = finite(x[rows, h])
                    held = int(scales[p, h, s, i]) if lead else 0
                    E = max(held, exponent(float(new.abs().max()), codes.dtype))
                    if lead and E > held:
                        ratio = 0.0 if held == 0 else 2.0 ** (held - E)
                        codes[p, h, s, i, :lead] = as_codes(rounded(numbers(codes[p, h, s, i, :lead]) * ratio, codes.dtype), codes.dtype)
                    unit = 2.0 ** (max(E, 1) - 127)
                    codes[p, h, s, i, lead:lead + len(rows)] = as_codes(rounded(new / unit, codes.dtype), codes.dtype)
                    scales[p, h, s, i] = E


def sequence(codes, scales, table, length):
    """K, V [H, length, D] in 64 bits of one sequence with page table row `table`."""
    S = codes.shape[2]
    ids = table[:-(-length // (16 * S))].long().to(codes.device)
    E = scales[ids].double()
    unit = torch.where(E > 0, torch.pow(torch.tensor(2.0, dtype=torch.float64), (E - 127).cpu()).to(E.device), 0.0)
    x = numbers(codes.view(torch.uint8)[ids].view(codes.dtype)) * unit[..., None, None]
    return tuple(x[:, :, :, i].transpose(0, 1).flatten(1, 3)[:, :length] for i in range(2))


def visible(length, window, sinks):
    t = torch.arange(length)
    return t if not window else t[(t < sinks) | (t >= length - window)]


def attention(q, k, v, sm_scale, cap=0.0):
    """q [Hq, D], k / v [H, tokens, D] in 64 bits -> o [Hq, D], lse [Hq], weights [Hq, tokens], and a bound of how far the kernels put a
    logit: 2^-21 of sum |q||k| for a sum of D products in a handful of steps of 24 bits and three roundings, and each channel of a query rounded by
    half a step of 2^-21 of the power of two that its row's largest has, 2^-22 of that at most."""
    H = len(k)
    group = q.shape[0] // H
    o, lse = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    p, off = torch.zeros(q.shape[0], k.shape[1], dtype=torch.float64, device=q.device), torch.zeros(q.shape[0], dtype=torch.float64, device=q.device)
    for h in range(q.shape[0] if k.shape[1] else 0):
        x = k[h // group] @ q[h].double() * sm_scale
        near, size = k[h // group].abs(), q[h].double().abs()
        off[h] = abs(sm_scale) * (2.0 ** -21 * (near @ size) + 2.0 ** -22 * size.max() * near.sum(1)).max()
        if cap:
            x = cap * torch.tanh(x / cap)
        p[h] = torch.softmax(x, 0)
        o[h], lse[h] = p[h] @ v[h // group], torch.logsumexp(x, 0)
    return o, lse, p, off


def evict(weight, length, budget, sinks, recent):
    """The places that one kv head keeps; weight [length], a list of numbers."""
    if length <= budget:
        return list(range(length))
    rest = [t for t in range(sinks, length - recent)]
    rest.sort(key=lambda t: (0, -weight[t], t) if not math.isnan(weight[t]) else (1, 0.0, t))
    return sorted(list(range(sinks)) + rest[:budget - sinks - recent] + list(range(length - recent, length)))


def move(codes, scales, weight, table, to_table, kept):
    """kept [b][h]: places, in a cache on the CPU, in place."""
    _, H, S, _, _, D = codes.shape
    page = 16 * S
    old_codes, old_scales, old_weight = codes.clone(), scales.clone(), weight.clone()
    for b in range(len(kept)):
        for h in range(H):
            for block in range(0, len(kept[b][h]), 16):
                src = kept[b][h][block:block + 16]
                p, s = int(to_table[b][block // page]), block // 16 % S
                at = [(int(table[b][t // page]), t % page // 16, t % 16, t % page) for t in src]
                for i, (sp, _, _, place) in enumerate(at):
                    weight[p, h, block % page + i] = old_weight[sp, h, place]
                for i in range(2):
                    held = [int(old_scales[sp, h, ss, i]) for sp, ss, _, _ in at]
                    E = max(held)
                    for j, (sp, ss, tau, _) in enumerate(at):
                        ratio = 0.0 if held[j] == 0 else 2.0 ** (held[j] - E)
                        x = numbers(old_codes[sp, h, ss, i, tau])
                        codes[p, h, s, i, j] = as_codes(x if held[j] == E and E else rounded(x * ratio, codes.dtype), codes.dtype)
                    scales[p, h, s, i] = E
