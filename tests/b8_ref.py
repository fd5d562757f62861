"""The 8-bit cache and the position rotation in plain torch on the CPU, from their definitions: tiles and codes, appending token by
token, the rotation in fp32 step by step and in 64 bits, attention in 64 bits with the error that a kernel's roundings may have."""
import math

import torch

LARGEST = {"e4m3": 448.0, "int8": 127.0}
RANGE = {"e4m3": (-15, 7), "int8": (-24, 9)}


def place(D):
    """(16, D): where channel c of a tile's token t lies in its row"""
    return torch.tensor([[(c // 16 ^ t % 8) * 16 + c % 16 for c in range(D)] for t in range(16)])


def pack(codes, exps):
    """codes (pages, heads, PS, D) uint8 in the order of the channels, exponents (pages, heads, PS / 16) -> cache bytes
    (pages, heads, PS, D + 1)"""
    P, H, PS, D = codes.shape
    t = torch.zeros((P, H, PS // 16, 16 * D + 16), dtype=torch.uint8)
    at = place(D).expand(P, H, PS // 16, 16, D)
    rows = torch.zeros((P, H, PS // 16, 16, D), dtype=torch.uint8).scatter_(-1, at, codes.view(P, H, PS // 16, 16, D))
    t[..., :16 * D] = rows.flatten(-2)
    t[..., 16 * D:16 * D + 4] = torch.ldexp(torch.ones(exps.shape), exps.float())[..., None].contiguous().view(torch.uint8)
    t[..., 16 * D + 4:] = 0xff                                 # (nothing reads these)
    return t.view(P, H, PS, D + 1)


def unpack(cache):
    """cache bytes -> (codes, scales (pages, heads, PS / 16) fp32, the unused bytes)"""
    P, H, PS, D1 = cache.shape
    D = D1 - 1
    t = cache.contiguous().view(P, H, PS // 16, 16 * D + 16)
    rows = t[..., :16 * D].reshape(P, H, PS // 16, 16, D)
    codes = rows.gather(-1, place(D).expand(rows.shape)).view(P, H, PS, D)
    return codes, t[..., 16 * D:16 * D + 4].contiguous().view(torch.float32)[..., 0], t[..., 16 * D + 4:]


def values(codes, fmt):
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).double()


def exponent(amax, fmt):
    lo, hi = RANGE[fmt]
    if amax == 0:
        return lo
    if math.isinf(amax):
        return hi
    e = lo
    while e < hi and amax > LARGEST[fmt] * 2.0 ** e:
        e += 1
    return e


def encode(y, fmt):
    """64-bit values -> codes: nearest, ties to even, the largest one beyond it; a NaN stays one (int8: 0)"""
    if fmt == "int8":
        return torch.nan_to_num(y, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return y.float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)      # (y: at most 24 bits, by a power of two)


def append(cache, key, value, slots, gk, gv, fmt):
    """the cache after a call that writes key / value (T, H, D) bf16 to the slots; runs of neighbours in one tile are one tile's tokens"""
    codes, scales, rest = unpack(cache)
    codes, scales = codes.clone(), scales.clone()
    P, H2, PS, D = codes.shape
    x = torch.cat((key.float() / gk[:, None], value.float() / gv[:, None]), 1)
    i = 0
    while i < len(slots):
        s = int(slots[i])
        if s < 0:
            i += 1
            continue
        j, rows = i, {}
        while j < len(slots) and int(slots[j]) >= 0 and int(slots[j]) // 16 == s // 16:
            rows[int(slots[j]) % 16] = j                       # (the last of a slot that is named twice)
            j += 1
        i = j
        page, sub = s // PS, s % PS // 16
        at, tok = list(rows), list(rows.values())
        for h in range(H2):
            y = x[tok, h].double()
            fin = torch.where(y.isnan(), 0.0, y.abs())
            e = exponent(float(fin.max()), fmt)
            old = None if 0 in rows else math.frexp(float(scales[page, h, sub]))[1] - 1
            if old is not None:
                e = max(e, old)
                if e > old:
                    keep = [r for r in range(16) if r not in rows]
                    c = codes[page, h, [sub * 16 + r for r in keep]]
                    codes[page, h, [sub * 16 + r for r in keep]] = encode(values(c, fmt) * 2.0 ** (old - e), fmt)
            codes[page, h, [sub * 16 + r for r in at]] = encode(y * 2.0 ** -e, fmt)
            scales[page, h, sub] = 2.0 ** e
    out = cache.clone().contiguous().view(P, H2, PS // 16, 16 * D + 16)
    rows = torch.zeros((P, H2, PS // 16, 16, D), dtype=torch.uint8)
    rows.scatter_(-1, place(D).expand(rows.shape), codes.view(rows.shape))
    out[..., :16 * D] = rows.flatten(-2)
    out[..., 16 * D:16 * D + 4] = scales[..., None].view(torch.uint8)
    return out.view(P, H2, PS, D + 1)


def turn(x, positions, table, interleaved, exact=False):
    """x (T, heads, D) bf16 turned by its positions: fp32 step by step, rounded to bf16, or (exact) in 64 bits with the sum of the
    products' magnitudes"""
    rot, t = table.shape[1], torch.float64 if exact else torch.float32
    cs = table[positions.clamp(0, table.shape[0] - 1)].to(t)[:, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    y = x.to(t)
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    out, mag = y.clone(), y.abs()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    if not exact:
        return out.to(torch.bfloat16)
    mag[..., a], mag[..., b] = (y[..., a] * c).abs() + (y[..., b] * s).abs(), (y[..., b] * c).abs() + (y[..., a] * s).abs()
    return out, mag


def sees(p, n, window, sinks):
    j = torch.arange(n)
    return (j <= p) & ((j > p - window) | (j < sinks) if window else torch.ones(n, dtype=torch.bool))


def attention(q, k, v, sm, window, sinks):
    """q (ql, H, G, D), k and v (L, H, D), 64 bits, the last ql tokens' rows. Returns the output, the log-sum-exp, the weights, and the
    score's error per unit of fp32 rounding: sum |q k| sm"""
    ql, H, G, D = q.shape
    L = k.shape[0]
    x = torch.einsum("thgd,jhd->hgtj", q, k) * sm
    mag = torch.einsum("thgd,jhd->hgtj", q.abs(), k.abs()) * abs(sm)
    see = torch.stack([sees(L - ql + t, L, window, sinks) for t in range(ql)])
    x = x.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(x, -1)
    w = torch.where(see, (x - torch.where(lse == -math.inf, 0.0, lse)[..., None]).exp(), 0.0)
    out = torch.einsum("hgtj,jhd->thgd", w, torch.nan_to_num(v, nan=0.0) if not v.isfinite().all() else v)
    reach = torch.where(see, mag, 0.0).amax(-1) if L else torch.zeros(H, G, ql, dtype=torch.float64)
    return out, lse, w, reach
